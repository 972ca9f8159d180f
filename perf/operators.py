"""Cases and plain forms of the paged KV-cache operators.

Three operators of a serving step over a cache kept in pages:

  write   rotate the new tokens' queries and keys (RoPE), quantise keys and values, store them in their pages
  read    the cached keys and values of whole sequences, back as contiguous FP16 rows
  attend  attention of the new tokens (a chunk of a prompt, or one token) over the pages

`run` computes them with elementary torch operations, or, where `own` is true, through atomflow_b200.ops.
"""
import math

import torch

own = False

DEV = "cuda"
ROPE_BASE = 500000.0
FORMATS = {"f16": torch.float16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}
# the largest code, and the largest scale whose product with it is a finite FP16 value
CODE_MAX = {"fp8": 448.0, "int8": 127.0}
SCALE_MAX = {"fp8": 146.125, "int8": 515.5}


def _case(name, op, fmt, heads, kv_heads, dim, page, seqs, q, kv, mix):
    return {"name": name, "op": op, "fmt": fmt, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "seqs": seqs, "q": q, "kv": kv, "mix": mix}


def listed():
    return [
        # one decoded token of one sequence: pure latency
        _case("write one token", "write", "fp8", 24, 8, 128, 16, 1, 1, 1025, "even"),
        # one decoded token of each sequence of a batch
        _case("write decode batch", "write", "int8", 32, 8, 128, 32, 64, 1, 700, "ragged"),
        # a batch of prompt chunks of the 8B-shaped model
        _case("write prompt chunks", "write", "fp8", 32, 8, 128, 64, 5, 2047, 2500, "ragged"),
        # a short sequence taken out of the cache
        _case("read short", "read", "int8", 24, 8, 128, 16, 1, 37, 37, "even"),
        # long sequences taken out of the cache, as when they are moved
        _case("read long", "read", "fp8", 32, 8, 128, 16, 12, 8191, 8191, "ragged"),
        # single-stream generation at position 1024 of the 3B-shaped model
        _case("attend one token", "attend", "f16", 24, 8, 128, 16, 1, 1, 1025, "even"),
        # single-stream generation far into a long document
        _case("attend long context", "attend", "fp8", 32, 8, 128, 64, 1, 1, 131001, "even"),
        # a decode batch at many different lengths
        _case("attend decode batch", "attend", "int8", 32, 8, 128, 16, 64, 1, 8000, "ragged"),
        # a decode batch of a model with small heads, a few drafted tokens each
        _case("attend drafts", "attend", "f16", 16, 4, 64, 32, 48, 4, 4099, "ragged"),
        # a whole prompt from an empty cache
        _case("attend prompt", "attend", "fp8", 24, 8, 128, 64, 1, 4096, 4096, "even"),
        # the next chunk of long prompts
        _case("attend chunks", "attend", "f16", 32, 8, 128, 16, 4, 1024, 16384, "even"),
        # chunks of some sequences beside single tokens of the others
        _case("attend mixed batch", "attend", "int8", 32, 4, 128, 128, 17, 385, 4097, "mixed"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        op = rng.choice(["write", "read", "attend", "attend"])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
        c = {"op": op, "fmt": rng.choice(list(FORMATS)), "heads": heads, "kv_heads": kv_heads,
             "dim": rng.choice([64, 128, 128]), "page": rng.choice([8, 16, 32, 64, 128]),
             "seqs": _spread(rng, 1, 64), "q": 1, "kv": 1, "mix": rng.choice(["even", "ragged", "mixed"])}
        if op == "read":
            c["kv"] = c["q"] = _spread(rng, 1, 8192)
        else:
            c["q"] = rng.choice([1, rng.randint(2, 16), _spread(rng, 17, 4096)])
            c["kv"] = c["q"] + (_spread(rng, 1, 32768) if op == "attend" else _spread(rng, 1, 1000))
        w = work(c)
        padded = c["seqs"] * heads * c["q"] * c["kv"]   # the plain form's scores
        tokens = c["seqs"] * c["kv"] * kv_heads * c["dim"]
        if w["flops"] <= 1.0e12 and w["bytes"] <= 4e8 and padded <= 2.0e9 and tokens <= 5e8:
            return c


def lengths(case):
    """New tokens and cached positions (the new tokens among them) of each sequence."""
    n, q, kv, mix = case["seqs"], case["q"], case["kv"], case["mix"]
    qs, kvs = [], []
    for b in range(n):
        part = ((b * 7) % n) / n   # 0 for the first sequence, spread over [0, 1)
        if case["op"] == "read":
            kvb = kv if mix == "even" else max(1, int(kv * (1 - 0.8 * part)))
            qs.append(kvb)
            kvs.append(kvb)
            continue
        qb = q if mix == "even" else max(1, int(q * (1 - 0.5 * part))) if mix == "ragged" else q if b % 4 == 0 else 1
        qs.append(qb)
        kvs.append(kv if mix == "even" else max(qb, int(kv * (1 - 0.8 * part))))
    return qs, kvs


def work(case):
    qs, kvs = lengths(case)
    h, g, d, t, n = case["heads"], case["kv_heads"], case["dim"], sum(qs), sum(kvs)
    row = g * (2 * d if case["fmt"] == "f16" else d + 2)   # one position's keys (or values) with their scales
    meta = 4 * (2 * len(qs) + 1 + sum(-(-v // case["page"]) for v in kvs))
    if case["op"] == "write":
        return {"bytes": 2 * t * (h + 2 * g) * d + 2 * t * h * d + 2 * t * row + 4 * t * d + meta, "flops": 3 * t * (h + g) * d}
    if case["op"] == "read":
        return {"bytes": 2 * n * row + 2 * n * g * d * 2 + meta, "flops": 2 * n * g * d}
    pairs = sum(q * kv - q * (q - 1) // 2 for q, kv in zip(qs, kvs))
    return {"bytes": 2 * n * row + 2 * 2 * t * h * d + meta, "flops": 4 * pairs * h * d}


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _quantise(x, fmt):
    """x float32 [..., dim] -> codes, FP16 scales: the scale is the smallest FP16 value that reaches the largest element."""
    top = x.abs().amax(dim=-1)
    want = top / CODE_MAX[fmt]
    scale = want.half()
    scale = torch.where(scale.float() < want, (scale.view(torch.int16) + 1).view(torch.float16), scale)
    scale = torch.where(top > 0, scale.clamp(max=SCALE_MAX[fmt]), torch.ones_like(scale))
    y = x / scale.float().unsqueeze(-1)
    y = y.clamp(-CODE_MAX[fmt], CODE_MAX[fmt])
    return (y.to(torch.float8_e4m3fn) if fmt == "fp8" else y.round().to(torch.int8)), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    qs, kvs = lengths(case)
    h, g, d, page, fmt, t = case["heads"], case["kv_heads"], case["dim"], case["page"], case["fmt"], sum(qs)
    counts = [-(-v // page) for v in kvs]
    used, width = sum(counts), max(counts)
    pages = used + 3
    places = torch.randperm(pages, generator=gen, device=DEV)[:used].to(torch.int32)
    table = torch.full((len(kvs), width), -1, dtype=torch.int32)
    at = torch.cat([torch.arange(c) + b * width for b, c in enumerate(counts)])
    table.view(-1)[at] = places.cpu()
    s = {"case": case, "block_table": table.to(DEV), "kv_len": torch.tensor(kvs, dtype=torch.int32, device=DEV),
         "cu_q": torch.tensor([0] + qs, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEV),
         "max_q": max(qs), "max_kv": max(kvs), "tokens": t}
    for name in ("k", "v"):
        x = _normal(gen, pages, page, g, d)
        if fmt == "f16":
            s[name + "_pages"], s[name + "_scale"] = x.half(), None
        else:
            s[name + "_pages"], s[name + "_scale"] = _quantise(x, fmt)
        del x
    if case["op"] == "write":
        s["qkv"] = _normal(gen, t, (h + 2 * g) * d).half()
        angle = torch.arange(max(kvs), device=DEV, dtype=torch.float64)[:, None] * (
            ROPE_BASE ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "attend":
        s["q"] = _normal(gen, t, h, d).half()
    return s


def run(state):
    if own:
        from atomflow_b200 import ops
        s = state
        pool = (s["k_pages"], s["v_pages"], s["block_table"], s["kv_len"], s["cu_q"])
        scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if s["case"]["op"] == "write":
            q = ops.paged_kv_write(s["qkv"], *pool, n_heads=s["case"]["heads"], cos=s["cos"], sin=s["sin"], **scales)
            return _written(s, q)
        if s["case"]["op"] == "read":
            return list(ops.paged_kv_read(*pool, s["tokens"], **scales))
        return [ops.paged_attention(s["q"], *pool, max_q=s["max_q"], max_kv=s["max_kv"], **scales)]
    return {"write": _write, "read": _read, "attend": _attend}[state["case"]["op"]](state)


def _written(s, q):
    return [q, s["k_pages"], s["v_pages"]] + ([] if s["k_scale"] is None else [s["k_scale"], s["v_scale"]])


def _tokens(s):
    """For each new token: its sequence, its place among the sequence's new tokens, its position in the cache."""
    t = torch.arange(s["tokens"], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["cu_q"][1:], t, right=True)
    i = t - s["cu_q"][b]
    return b, i, s["kv_len"][b] - (s["cu_q"][b + 1] - s["cu_q"][b]) + i


def _rotate(x, c, s):
    """Pair (j, j + dim/2) of x FP16 by its angle, in 64 bits up to the one rounding of y*s that the framework's rotation has."""
    x, y = x.double().chunk(2, dim=-1)
    c, s = c.double().unsqueeze(1), s.double().unsqueeze(1)
    lo = x * c - (y * s).float().double()
    hi = x * s + (y * c).float().double()
    return torch.cat([lo, hi], dim=-1).float().half()


def _write(s):
    case = s["case"]
    h, g, d, page, fmt = case["heads"], case["kv_heads"], case["dim"], case["page"], case["fmt"]
    b, _, pos = _tokens(s)
    x = s["qkv"].view(-1, h + 2 * g, d)
    r = _rotate(x[:, :h + g], s["cos"][pos], s["sin"][pos])
    at = (s["block_table"][b, pos // page].long(), (pos % page).long())
    for name, new in (("k", r[:, h:]), ("v", x[:, h + g:])):
        pool, scale = s[name + "_pages"], s[name + "_scale"]
        if fmt == "f16":
            pool[at] = new
            continue
        code, sc = _quantise(new.float(), fmt)
        pool.view(torch.uint8)[at] = code.view(torch.uint8)
        scale[at] = sc
    return _written(s, r[:, :h].contiguous())


def _gather(s, name, at):
    """Cached values at pages and slots, in 32 bits."""
    pool, scale = s[name + "_pages"], s[name + "_scale"]
    if scale is None:
        return pool[at].float()
    return pool.view(torch.uint8)[at].view(pool.dtype).float() * scale[at].float().unsqueeze(-1)


def _read(s):
    b, _, pos = _tokens(s)
    page = s["case"]["page"]
    at = (s["block_table"][b, pos // page].long(), (pos % page).long())
    return [_gather(s, name, at).half() for name in ("k", "v")]


def _attend(s):
    case = s["case"]
    h, g, d, page, n, mq, mk = case["heads"], case["kv_heads"], case["dim"], case["page"], case["seqs"], s["max_q"], s["max_kv"]
    b, i, _ = _tokens(s)
    j = torch.arange(mk, device=DEV)
    at = (s["block_table"][:, j // page].clamp(min=0).long(), (j % page).expand(n, mk))
    inside = (j < s["kv_len"][:, None])[:, :, None, None]
    k = (_gather(s, "k", at) * inside).permute(0, 2, 3, 1)            # [n, g, d, mk]
    v = (_gather(s, "v", at) * inside).permute(0, 2, 1, 3)            # [n, g, mk, d]
    ql = s["cu_q"][1:] - s["cu_q"][:-1]
    rows = (s["cu_q"][:-1, None] + torch.arange(mq, device=DEV)).clamp(max=s["tokens"] - 1).long()
    q = s["q"][rows].float().view(n, mq, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(n, g, -1, d)
    score = torch.matmul(q, k).view(n, g, h // g, mq, mk).mul_(1 / math.sqrt(d))
    seen = j < ((s["kv_len"] - ql)[:, None] + torch.arange(mq, device=DEV) + 1)[:, :, None]   # [n, mq, mk]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(n, g, -1, mk), v).view(n, g, h // g, mq, d) / torch.where(total > 0, total, 1.0)
    return [o.permute(0, 3, 1, 2, 4)[b, i.long()].reshape(-1, h, d).half()]


def exact(case, seed):
    """The definitions, sequence by sequence, in 64 bits."""
    s = prepare(case, seed)
    qs, kvs = lengths(case)
    h, g, d, page, fmt = case["heads"], case["kv_heads"], case["dim"], case["page"], case["fmt"]
    table = s["block_table"].cpu().long()

    def slots(b, first, count):
        p = torch.arange(first, first + count)
        return (table[b, p // page] * page + p % page).to(DEV)

    def cached(name, where, head):
        x = s[name + "_pages"].view(-1, g, d)[:, head]
        x = (x.view(torch.uint8)[where].view(x.dtype) if fmt == "fp8" else x[where]).double()
        return x if fmt == "f16" else x * s[name + "_scale"].view(-1, g)[where, head].double().unsqueeze(-1)

    if case["op"] == "read":
        return [torch.cat([torch.stack([cached(name, slots(b, 0, n), e) for e in range(g)], dim=1)
                           for b, n in enumerate(kvs)]) for name in ("k", "v")]
    if case["op"] == "write":
        place = torch.cat([torch.arange(n - m, n) for m, n in zip(qs, kvs)]).to(DEV)
        where = torch.cat([slots(b, n - m, m) for b, (m, n) in enumerate(zip(qs, kvs))])
        x = s["qkv"].double().view(-1, h + 2 * g, d)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[place][:, None]
        z = torch.complex(x[:, :h + g, :d // 2], x[:, :h + g, d // 2:]) * turn
        r = torch.cat([z.real, z.imag], dim=-1)
        out, scales = [r[:, :h]], []
        for name, new in (("k", r[:, h:]), ("v", x[:, h + g:])):
            pool = s[name + "_pages"].double()
            if fmt != "f16":
                scale = s[name + "_scale"].double()
                step = new.abs().amax(dim=-1) / CODE_MAX[fmt]
                scale.view(-1, g)[where] = step
                scales.append(scale)
                new = new / step.unsqueeze(-1)
            pool.view(-1, g, d)[where] = new
            out.append(None if fmt == "int8" else pool)
        return out + scales
    pieces, row = [], 0
    for b, (m, n) in enumerate(zip(qs, kvs)):
        where = slots(b, 0, n)
        part = torch.empty(m, h, d, dtype=torch.float64, device=DEV)
        hidden = torch.arange(n, device=DEV)[None] > torch.arange(n - m, n, device=DEV)[:, None]
        for head in range(h):
            k, v = (cached(name, where, head // (h // g)) for name in ("k", "v"))
            w = s["q"][row:row + m, head].double() @ k.T / d ** 0.5
            part[:, head] = torch.softmax(w.masked_fill_(hidden, -math.inf), dim=-1) @ v
        pieces.append(part)
        row += m
    return [torch.cat(pieces)]
