"""The paged KV cache on the GPU: write, read and attention against plain 64-bit
forms (numpy on the host for what is exact, torch float64 for attention), at the
sizes, masks and layouts where they can go wrong.

Tolerance of attention, per output element, with p_j the exact weights (sum 1),
W = sum p_j |v_j| and w_j = exp(s_j - max s) the weights before the division:
  * the output's FP16 rounding: 2^-11 |out| + 2^-25 (subnormal)
  * P is rounded to FP16 before the product: 2^-11 W, and 2^-25 per weight that
    is subnormal in FP16, relative to a largest weight of at least 1:
    2^-25 sum |v_j| / sum w_j
  * 8-bit caches: the codes are exact in FP16, K's scale multiplies S in FP32, and
    V's goes into the one rounding of P (less a power of two, exact in FP16 with the
    codes, or brought to about 1 for the largest; a weight that is then subnormal is
    off by 2^-25 of the largest scale's: 2^-25 n max|v| / sum w_j)
  * scores, sums and products in FP32: a score error of 2^-24 (HD / 16 + 8) scale
    sum |q_d k_d| and of 2^-22 relative in each exponential's argument and
    value, and 2^-19 W for the sums (up to 2^4 partial orders, truncating
    accumulation)
  a score error of at most d changes every normalised weight by at most a factor
  exp(2 d), so out by (exp(2 d) - 1) W.
"""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FMT = {"f16": torch.float16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"fp8": np.float32(448), "int8": np.float32(127)}
CAP = {"fp8": np.float16(146.125), "int8": np.float16(515.5)}
DEV = "cuda"


def faults(clear=True):
    from atomflow_b200 import lib
    torch.cuda.synchronize()
    v = ctypes.c_uint(0)
    assert lib().af_device_faults(ctypes.byref(v), 1 if clear else 0) == 0
    return v.value


def quantise(x, fmt):
    """x float32 numpy [..., hd] -> codes (uint8 bits), scales float16, by the definition."""
    amax = np.abs(x).max(-1)
    want = (amax / TOP[fmt]).astype(np.float32)
    with np.errstate(over="ignore"):
        s = want.astype(np.float16)
    s = np.where(s.astype(np.float32) < want, np.nextafter(s, np.float16(np.inf)), s)
    s = np.where(amax > 0, np.minimum(s, CAP[fmt]), np.float16(1)).astype(np.float16)
    y = x / s.astype(np.float32)[..., None]
    if fmt == "int8":
        return np.rint(np.clip(y, -127, 127)).astype(np.int8).view(np.uint8), s
    y = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn)
    return y.view(torch.uint8).numpy(), s


class Cache:
    """A pool with every byte poisoned (NaN where the format has one), and a batch over it."""

    def __init__(self, fmt, kv_len, q_len, nkv=2, hd=128, page=16, seed=0, spare=3, k=None, v=None, page_pad=0):
        g = torch.Generator().manual_seed(seed)
        self.fmt, self.nkv, self.hd, self.page = fmt, nkv, hd, page
        counts = [-(-n // page) for n in kv_len]
        used, width = sum(counts), max(counts + [1])
        n_pages = used + spare
        perm = torch.randperm(n_pages, generator=g)[:used].tolist()
        table = torch.full((len(kv_len), width), -7, dtype=torch.int32)
        at = 0
        for b, c in enumerate(counts):
            table[b, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
            at += c
        raw = (n_pages, page + page_pad, nkv, hd)
        poison = {"f16": float("nan"), "int8": -128, "fp8": 0x7f}[fmt]
        dt = {"f16": torch.float16, "int8": torch.int8, "fp8": torch.uint8}[fmt]
        self.k = torch.full(raw, poison, dtype=dt).to(DEV)[:, :page]
        self.v = torch.full(raw, poison, dtype=dt).to(DEV)[:, :page]
        if fmt == "fp8":
            self.k, self.v = self.k.view(torch.float8_e4m3fn), self.v.view(torch.float8_e4m3fn)
        self.ks = self.vs = None
        if fmt != "f16":
            self.ks = torch.full((n_pages, page + page_pad, nkv), float("nan"), dtype=torch.float16, device=DEV)[:, :page]
            self.vs = self.ks.clone()[:, :page] if not page_pad else torch.full_like(self.ks.as_strided(
                (n_pages, page + page_pad, nkv), ((page + page_pad) * nkv, nkv, 1)), float("nan"))[:, :page]
        self.table = table.to(DEV)
        self.kv_len, self.q_len = list(kv_len), list(q_len)
        self.len_t = torch.tensor(kv_len, dtype=torch.int32, device=DEV)
        self.cu = torch.tensor([0] + list(np.cumsum(q_len)), dtype=torch.int32, device=DEV)
        self.T = sum(q_len)
        for b, n in enumerate(kv_len):   # contents by plain indexing
            kk = torch.randn(n, nkv, hd, generator=g) if k is None else k[b]
            vv = torch.randn(n, nkv, hd, generator=g) if v is None else v[b]
            self.put(b, 0, kk, vv)

    def where(self, b, first, count):
        p = torch.arange(first, first + count, device=DEV)
        return self.table[b, p // self.page].long(), p % self.page

    def put(self, b, first, k, v):
        at = self.where(b, first, k.shape[0])
        for pool, scale, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
            if self.fmt == "f16":
                pool[at] = x.to(torch.float16).to(DEV)
            else:
                code, s = quantise(x.to(torch.float16).float().numpy(), self.fmt)
                pool.view(torch.uint8)[at] = torch.from_numpy(code).to(DEV)
                scale[at] = torch.from_numpy(s).to(DEV)

    def values(self, b, first=0, count=None):
        """float64 [count, nkv, hd] k, v as the codes and scales say."""
        at = self.where(b, first, self.kv_len[b] - first if count is None else count)
        out = []
        for pool, scale in ((self.k, self.ks), (self.v, self.vs)):
            if self.fmt == "f16":
                out.append(pool[at].double())
            else:
                x = pool.view(torch.uint8)[at].view(FMT[self.fmt])
                out.append((x.float() if self.fmt == "fp8" else x).double() * scale[at].double()[..., None])
        return out

    @property
    def args(self):
        return self.k, self.v, self.table, self.len_t, self.cu

    @property
    def scales(self):
        return dict(k_scale=self.ks, v_scale=self.vs)


def attention_f64(c, q, scale, b, row):
    """(out, tolerance) float64 [q_len, nh, hd] of sequence b."""
    m, n, nh, hd = c.q_len[b], c.kv_len[b], q.shape[1], c.hd
    k, v = (x.repeat_interleave(nh // c.nkv, dim=1).transpose(0, 1) for x in c.values(b))   # [nh, n, hd]
    x = q[row:row + m].double().transpose(0, 1)                                               # [nh, m, hd]
    hidden = (torch.arange(n, device=DEV)[None] > torch.arange(n - m, n, device=DEV)[:, None])
    s = (x @ k.transpose(1, 2) * scale).masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True) if n else s.new_full((nh, m, 1), -math.inf)
    w = torch.exp(s - torch.where(top > -math.inf, top, 0.0)).masked_fill(hidden, 0.0)
    total = w.sum(-1, keepdim=True)
    p = w / total.clamp(min=1e-300)
    out = p @ v
    W = p @ v.abs()
    absqk = (x.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(hidden, 0.0).amax(-1, keepdim=True) if n else top * 0
    d = absqk * (2.0 ** -24 * (hd / 16 + 8)) + 2.0 ** -22 * (s.masked_fill(hidden, 0.0).abs().amax(-1, keepdim=True) + 1 if n else 1)
    quant = c.fmt != "f16"
    seen = (~hidden).double()
    tol = (2.0 ** -11 * out.abs() + 2.0 ** -25 + W * (2.0 ** -11 + torch.expm1(2 * d) + 2.0 ** -19) +
           2.0 ** -25 * (seen @ v.abs()) / total.clamp(min=1e-300).clamp(min=1.0))
    if quant:
        tol = tol + 2.0 ** -25 * (seen @ v.abs().amax(-1, keepdim=True)) / total.clamp(min=1e-300).clamp(min=1.0)
    empty = total == 0
    out, tol = out.masked_fill(empty, 0.0), tol.masked_fill(empty, 0.0)
    return out.transpose(0, 1), tol.transpose(0, 1)


def check_attention(c, nh, seed=1, scale=None, q=None, tail=2, **kw):
    from atomflow_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(seed)
    if q is None:
        q = torch.randn(c.T + tail, nh, c.hd, generator=g, device=DEV).half()
    out = torch.full(q.shape, 77.0, dtype=torch.float16, device=DEV)
    got = ops.paged_attention(q, *c.args, scale=scale, out=out, **c.scales, **kw)
    assert got is out and faults() == 0
    scale = c.hd ** -0.5 if scale is None else scale
    row = 0
    for b, m in enumerate(c.q_len):
        if m:
            want, tol = attention_f64(c, q, scale, b, row)
            err = (got[row:row + m].double() - want).abs()
            bad = ~(err <= tol)
            assert not bad.any(), (b, int(bad.sum()), bad.nonzero()[:4].tolist(), float((err / tol).nan_to_num(nan=9e9).max()))
        row += m
    assert (got[row:] == 77.0).all()   # rows of no sequence: as they were
    return q, got


# ------------------------------------------------------------------ write
def qkv_rows(T, nh, nkv, hd, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, (nh + 2 * nkv) * hd + pad, generator=g).half()
    return x.to(DEV)[:, :(nh + 2 * nkv) * hd] if pad else x.to(DEV)


def rope_tables(n, hd):
    from atomflow_b200 import lib
    c, s = np.zeros((n, hd // 2), np.float32), np.zeros((n, hd // 2), np.float32)
    assert lib().af_rope_tables(c.ctypes.data, s.ctypes.data, n, hd, 500000.0) == 0
    return torch.from_numpy(c).to(DEV), torch.from_numpy(s).to(DEV)


def rope_np(x, c, s):
    """The framework's rotation in exact arithmetic up to its own two roundings (float64 holds the products exactly)."""
    x = x.astype(np.float64)
    c, s = c.astype(np.float64)[:, None], s.astype(np.float64)[:, None]
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    lo = a * c - (b * s).astype(np.float32).astype(np.float64)
    hi = a * s + (b * c).astype(np.float32).astype(np.float64)
    return np.concatenate([lo, hi], -1).astype(np.float32).astype(np.float16)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("hd,nkv,nh,page", [(128, 8, 24, 16), (64, 1, 5, 8), (128, 3, 3, 256), (64, 7, 0, 64)])
@pytest.mark.parametrize("rotate", [True, False])
def test_write(fmt, hd, nkv, nh, page, rotate):
    from atomflow_b200 import ops
    kv, ql = [70, 5, 1, 0, 33, 300], [3, 5, 1, 0, 33, 1]
    c = Cache(fmt, kv, ql, nkv, hd, page, seed=3)
    before = [t.clone() if t is not None else None for t in (c.k, c.v, c.ks, c.vs)]
    T = c.T + 3
    qkv = qkv_rows(T, nh, nkv, hd, 4, pad=8)
    keep = qkv.clone()
    kw = {}
    if rotate:
        kw = dict(zip(("cos", "sin"), rope_tables(300, hd)))
        if nh:
            kw["q_out"] = torch.full((T, nh, hd), 5.0, dtype=torch.float16, device=DEV)
    q = ops.paged_kv_write(qkv, *c.args, n_heads=nh, **c.scales, **kw)
    assert faults() == 0 and torch.equal(qkv, keep)
    x = keep.cpu().numpy().reshape(T, nh + 2 * nkv, hd)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(kv, ql)])
    r = x[:c.T].copy()
    if rotate:
        cs, sn = (kw[k].cpu().numpy()[pos] for k in ("cos", "sin"))
        r[:, :nh + nkv] = rope_np(r[:, :nh + nkv], cs, sn)
    if nh:
        assert np.array_equal(q[:c.T].cpu().numpy(), r[:, :nh])
        if rotate:
            assert (q[c.T:] == 5.0).all()
    want = Cache(fmt, kv, ql, nkv, hd, page, seed=3)   # the same pool, the new rows put in by plain indexing
    row = 0
    for b, m in enumerate(ql):
        if m:
            want.put(b, kv[b] - m, torch.from_numpy(r[row:row + m, nh:nh + nkv]), torch.from_numpy(r[row:row + m, nh + nkv:]))
        row += m
    bits = lambda t: t.contiguous().view(torch.uint8) if t.dtype != torch.float16 else t.contiguous().view(torch.int16)
    for got, ref, old in zip((c.k, c.v, c.ks, c.vs), (want.k, want.v, want.ks, want.vs), before):
        if got is not None:
            assert torch.equal(bits(got), bits(ref)) and not torch.equal(bits(got), bits(old))


def test_write_holds_the_one_sequence_cache_rows():
    """FP16 pages hold, bit for bit, the rows that af_rope_kv_write puts into the contiguous cache; q alike."""
    from atomflow_b200 import lib, ops
    nh, nkv, hd, n = 6, 2, 128, 40
    cos, sin = rope_tables(64, hd)
    qkv = qkv_rows(n, nh, nkv, hd, 9)
    c = Cache("f16", [n], [n], nkv, hd, 8)
    q = ops.paged_kv_write(qkv, *c.args, n_heads=nh, cos=cos, sin=sin)
    kc = torch.zeros(64, nkv * hd, dtype=torch.float16, device=DEV)
    vc = torch.zeros_like(kc)
    one = qkv.clone()
    st = torch.cuda.current_stream().cuda_stream
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    for i in range(n):
        assert lib().af_rope_kv_write(one[i].data_ptr(), cos.data_ptr(), sin.data_ptr(), pos[i:].data_ptr(), kc.data_ptr(),
                                      vc.data_ptr(), nh, nkv, hd, 64, st) == 0
    k, v = c.values(0)
    assert torch.equal(k.half().reshape(n, -1), kc[:n]) and torch.equal(v.half().reshape(n, -1), vc[:n])
    assert torch.equal(q.reshape(n, -1), one[:, :nh * hd]) and faults() == 0


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_write_extreme_values(fmt):
    """Vectors of zeros, of subnormals, of the largest values, with infinities and NaN."""
    from atomflow_b200 import ops
    hd, rows = 64, []
    g = torch.Generator().manual_seed(0)
    for scale in (0.0, 6e-8, 1e-6, 2e-5, 1e-3, 1.0, 300.0, 65504.0):
        rows.append((torch.rand(hd, generator=g) * 2 - 1) * scale)
    for v in (65504.0, -65504.0, 6e-8):
        rows.append(torch.full((hd,), v))
    x = torch.stack(rows).half()
    n = x.shape[0]
    c = Cache(fmt, [n], [n], 1, hd, 8)
    ops.paged_kv_write(torch.cat([x, x], 1).to(DEV), *c.args, n_heads=0, **c.scales)
    k, v = c.values(0)
    code, s = quantise(x.float().numpy(), fmt)
    at = c.where(0, 0, n)
    assert torch.equal(c.k.view(torch.uint8)[at][:, 0].cpu(), torch.from_numpy(code))
    assert torch.equal(c.ks[at][:, 0].cpu(), torch.from_numpy(s)) and torch.equal(k, v)
    # half a step of the code, the largest value within the scale's cap
    err = (k[:, 0].cpu() - x.double()).abs()
    sc = torch.from_numpy(s.astype(np.float64))[:, None]
    half = 0.5 * sc if fmt == "int8" else torch.maximum(x.double().abs() * 2.0 ** -4, sc * 2.0 ** -10)
    assert (err <= half * (1 + 2.0 ** -20)).all()
    kr, vr = ops.paged_kv_read(*c.args, n, **c.scales)
    assert torch.isfinite(kr).all() and faults() == 0
    # an infinity takes the largest code; NaN is E4M3's NaN, INT8's 0; the other elements are not touched by a NaN
    y = torch.ones(2, hd)
    y[0, 3], y[0, 4], y[1, 5] = math.inf, -math.inf, math.nan
    c = Cache(fmt, [2], [2], 1, hd, 8)
    ops.paged_kv_write(torch.cat([y, y], 1).half().to(DEV), *c.args, n_heads=0, **c.scales)
    kr = ops.paged_kv_read(*c.args, 2, **c.scales)[0][:, 0].cpu()
    big = np.float16(np.float32(TOP[fmt]) * np.float32(CAP[fmt]))
    assert kr[0, 3] == float(big) and kr[0, 4] == -float(big)
    assert (kr[1, 5].isnan() if fmt == "fp8" else kr[1, 5] == 0) and abs(float(kr[1, 6]) - 1.0) <= 2.0 ** -4


def test_write_skips_what_has_no_place():
    """Positions past the tables, before the cache, pages outside the pool, sequences that leave the buffers."""
    from atomflow_b200 import ops
    nkv, hd = 1, 64
    cos, sin = rope_tables(20, hd)
    c = Cache("f16", [20, 40, 2, 9], [2, 3, 5, 1], nkv, hd, 8, seed=2)
    c.table[3, 1] = 10 ** 6                 # sequence 3's position 8
    qkv = qkv_rows(c.T, 1, nkv, hd, 1)
    old = c.k.clone()
    q = torch.full((c.T, 1, hd), 3.0, dtype=torch.float16, device=DEV)
    ops.paged_kv_write(qkv, *c.args, n_heads=1, cos=cos, sin=sin, q_out=q)
    assert faults() == 2 | 16               # position past the tables; bad page
    changed = {(int(p), int(s)) for p, s in ((c.k.view(torch.int16) != old.view(torch.int16)).any(-1).any(-1)).nonzero().tolist()}
    at = [c.where(0, 18, 2), c.where(2, 0, 2)]
    assert changed == {(int(p), int(s)) for a in at for p, s in zip(*a)}
    assert [bool((q[i] == 3.0).all()) for i in range(c.T)] == [False] * 2 + [True] * 3 + [True] * 3 + [False] * 2 + [True]
    bad = c.cu.clone()
    bad[-1] = c.T + 50                      # the last sequence's rows leave the buffers
    before = c.k.clone()
    ops.paged_kv_write(qkv, c.k, c.v, c.table, c.len_t, bad, n_heads=1)
    f = faults()
    assert f == 16
    new = (c.k.view(torch.int16) != before.view(torch.int16)).any(-1).any(-1).nonzero().tolist()
    ok = {(int(p), int(s)) for a in (c.where(0, 18, 2), c.where(1, 37, 3), c.where(2, 0, 2)) for p, s in zip(*a)}
    assert {(a, b) for a, b in new} <= ok


# ------------------------------------------------------------------- read
@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("hd,nkv,page", [(128, 8, 16), (64, 3, 8), (128, 1, 128)])
def test_read(fmt, hd, nkv, page):
    from atomflow_b200 import ops
    kv, ql = [70, 5, 1, 0, 129, 2], [70, 2, 1, 0, 64, 5]    # whole, the last rows, more than there are
    c = Cache(fmt, kv, ql, nkv, hd, page, seed=5)
    out = [torch.full((c.T + 5, nkv, hd), 9.0, dtype=torch.float16, device=DEV) for _ in range(2)]
    k, v = ops.paged_kv_read(*c.args, c.T + 5, k_out=out[0], v_out=out[1], **c.scales)
    assert k is out[0] and v is out[1] and faults() == 0
    row = 0
    for b, (n, m) in enumerate(zip(kv, ql)):
        none = max(0, m - n)
        for got, want in zip((k, v), c.values(b, n - (m - none))):
            assert (got[row:row + none] == 0).all()
            assert torch.equal(got[row + none:row + m], want.half())
        row += m
    assert (k[row:] == 9.0).all() and (v[row:] == 9.0).all()
    k2, v2 = ops.paged_kv_read(*c.args, c.T, **c.scales)
    assert torch.equal(k2, k[:c.T]) and torch.equal(v2, v[:c.T])
    c.table[4, 70 // page] = c.k.shape[0]       # a page outside the pool: zeros, the others stay
    k3, _ = ops.paged_kv_read(*c.args, c.T, **c.scales)
    assert faults() == 16
    assert torch.equal(k3[:73], k[:73])


# -------------------------------------------------------------- attention
GROUPS = [(8, 8), (3, 1), (8, 2), (10, 2), (16, 2)]


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", GROUPS)
def test_single_tokens(fmt, hd, nh, nkv):
    c = Cache(fmt, [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 400, 0], [1] * 11 + [0], nkv, hd, 16)
    check_attention(c, nh, max_q=1, max_kv=400)
    check_attention(c, nh)                                   # no bounds: both kernels run


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv,ql", [(4, 4, 16), (8, 2, 4), (6, 2, 5), (16, 2, 2), (5, 1, 3)])
def test_few_rows(fmt, hd, nh, nkv, ql):
    """Up to 16 rows per kv head, with rows that do not see the last positions."""
    kv = [ql, ql + 1, 40, 129, 500]
    c = Cache(fmt, kv, [ql] * len(kv), nkv, hd, 8)
    check_attention(c, nh, max_q=ql, max_kv=500)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", GROUPS)
def test_chunks(fmt, hd, nh, nkv):
    c = Cache(fmt, [130, 128, 127, 300, 385], [130, 20, 127, 43, 129], nkv, hd, 32)
    check_attention(c, nh, max_q=130, max_kv=385)


@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_pages_of_every_size(fmt, page):
    c = Cache(fmt, [page - 1, page, page + 1, 3 * page + 5, 700], [1, 3, page, 60, 1], 2, 128, page)
    check_attention(c, 4)


@pytest.mark.parametrize("fmt", list(FMT))
def test_mixed_batch(fmt):
    """Chunks beside single tokens, empty sequences between them, a chunk longer than its cache."""
    kv, ql = [500, 1, 0, 77, 300, 20, 900, 3], [200, 1, 0, 1, 300, 33, 2, 0]
    c = Cache(fmt, kv, ql, 2, 128, 16)
    _, got = check_attention(c, 8, max_q=300, max_kv=900)
    first = 200 + 1 + 1 + 300
    assert (got[first:first + 13] == 0).all()                # rows before position 0
    check_attention(c, 32, max_q=300, max_kv=900)


@pytest.mark.parametrize("ql", [1, 3, 64])
def test_rows_that_see_nothing(ql):
    c = Cache("f16", [0, 0, 1], [ql, ql, ql], 2, 128, 16)
    check_attention(c, 4, max_q=ql, max_kv=16)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("ql,kv", [(1, 40000), (2, 9000), (64, 20000), (200, 5000)])
def test_long_caches_split_over_a_cluster(fmt, ql, kv):
    """One sequence, one kv head: the positions are split; the bits do not depend on the run."""
    from atomflow_b200 import ops
    c = Cache(fmt, [kv], [ql], 1, 128, 64)
    q, got = check_attention(c, 4, max_q=ql, max_kv=kv, tail=0)
    again = ops.paged_attention(q, *c.args, max_q=ql, max_kv=kv, **c.scales)
    assert torch.equal(got, again)
    # the bounds choose the split, not the meaning
    check_attention(c, 4, max_q=ql, max_kv=1, tail=0)


@pytest.mark.parametrize("ql", [1, 100])
def test_large_scores(ql):
    """Scores far apart, rising along the cache (the running maximum moves in every tile) and falling."""
    n, hd = 1000, 128
    for sign in (1, -1):
        ramp = torch.linspace(-8, 8, n)[:, None, None] * sign
        k = [ramp.expand(n, 1, hd) + 0.05 * torch.randn(n, 1, hd, generator=torch.Generator().manual_seed(1))]
        c = Cache("f16", [n], [ql], 1, hd, 16, k=k)
        q = torch.ones(ql, 4, hd, dtype=torch.float16, device=DEV)
        check_attention(c, 4, q=q)
        check_attention(c, 4, scale=1.0, q=q)
        check_attention(c, 4, scale=1e-4, q=q)


@pytest.mark.parametrize("fmt", list(FMT))
def test_strides(fmt):
    """Pages that interleave with another pool's, q inside the packed projection, padded rows of the table."""
    from atomflow_b200 import ops
    c = Cache(fmt, [50, 300, 7], [1, 40, 7], 2, 64, 16, page_pad=16)
    wide = torch.full((3, c.table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide[:, :c.table.shape[1]]
    qkv = qkv_rows(c.T, 4, 2, 64, 3, pad=16)
    q = ops.paged_kv_write(qkv, *c.args, n_heads=4, **c.scales)
    assert q.data_ptr() == qkv.data_ptr() and q.shape == (c.T, 4, 64) and not q.is_contiguous()
    check_attention(c, 4, q=q)
    check_attention(c, 4, q=q, max_q=40)
    k, v = ops.paged_kv_read(*c.args, c.T, **c.scales)
    row = 0
    for b, m in enumerate(c.q_len):
        for got, want in zip((k, v), c.values(b, c.kv_len[b] - m)):
            assert torch.equal(got[row:row + m], want.half())
        row += m


@pytest.mark.parametrize("ql", [1, 40])
def test_offsets_past_32_bits(ql):
    """Pages more than 4 GB (and 2^31 elements) into the pool."""
    from atomflow_b200 import ops
    nkv, hd, page = 8, 128, 128
    n_pages = 20000                                           # 262,144 bytes each: 5.2 GB
    k = torch.empty(n_pages, page, nkv, hd, dtype=torch.float16, device=DEV)
    v = torch.empty(n_pages, page, nkv, hd, dtype=torch.float16, device=DEV)
    kv = 300
    table = torch.tensor([[19999, 16500, 3]], dtype=torch.int32, device=DEV)
    c = Cache("f16", [kv], [ql], nkv, hd, page)
    for i in range(3):
        k[int(table[0, i])], v[int(table[0, i])] = c.k[int(c.table[0, i])], c.v[int(c.table[0, i])]
    c.k, c.v, c.table = k, v, table
    check_attention(c, nkv)
    qkv = qkv_rows(ql, 0, nkv, hd, 1)
    ops.paged_kv_write(qkv, *c.args, n_heads=0)
    got = ops.paged_kv_read(*c.args, ql)
    x = qkv.view(ql, 2 * nkv, hd)
    assert torch.equal(got[0], x[:, :nkv]) and torch.equal(got[1], x[:, nkv:]) and faults() == 0


@pytest.mark.parametrize("ql", [1, 40])
@pytest.mark.parametrize("fmt", ["f16", "fp8"])
def test_bad_pages_and_sequences_touch_no_other(ql, fmt):
    from atomflow_b200 import ops
    c = Cache(fmt, [200] * 4, [ql] * 4, 2, 128, 16)
    q, good = check_attention(c, 8, max_q=ql, tail=0)
    keep = c.table.clone()
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        c.table = keep.clone()
        c.table[1, 3] = bad
        out = ops.paged_attention(q, *c.args, max_q=ql, **c.scales)
        assert faults() == 16
        for b in (0, 2, 3):
            assert torch.equal(out[b * ql:(b + 1) * ql], good[b * ql:(b + 1) * ql])
    c.table = keep
    for lens in ([200, 209, 200, 200], [200, -1, 200, 200]):   # more positions than pages; negative
        out = torch.full_like(q, 4.0)
        t = torch.tensor(lens, dtype=torch.int32, device=DEV)
        ops.paged_attention(q, c.k, c.v, c.table, t, c.cu, max_q=ql, out=out, **c.scales)
        assert faults() == 16 and (out[ql:2 * ql] == 4.0).all() and torch.equal(out[2 * ql:], good[2 * ql:])
    cu = c.cu.clone()
    cu[-1] = 10 ** 6
    out = torch.full_like(q, 4.0)
    ops.paged_attention(q, c.k, c.v, c.table, c.len_t, cu, max_q=ql, out=out, **c.scales)
    assert faults() == 16 and (out[3 * ql:] == 4.0).all() and torch.equal(out[:3 * ql], good[:3 * ql])


def test_a_bound_that_does_not_hold_is_recorded():
    from atomflow_b200 import ops
    c = Cache("f16", [50, 50], [1, 30], 1, 128, 16)
    q = torch.randn(31, 4, 128, device=DEV).half()
    out = torch.full_like(q, 4.0)
    ops.paged_attention(q, *c.args, max_q=1, out=out)
    assert faults() == 16 and (out[1:] == 4.0).all() and not (out[0] == 4.0).all()
    check_attention(c, 4, max_q=20)                          # too low a bound above the few rows does no harm


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_graph_replay_follows_the_arrays(fmt):
    """One captured step (write, attend) replays with other lengths, rows and pages; two graphs run at once."""
    from atomflow_b200 import ops
    nkv, hd, nh = 2, 128, 8
    cos, sin = rope_tables(600, hd)
    shapes = [([100, 300, 41], [1, 1, 1]), ([17, 500, 200], [1, 0, 2]), ([513, 30, 64], [1, 1, 1])]
    graphs = []
    for i, (kv, ql) in enumerate(shapes[:2]):
        c = Cache(fmt, [513, 513, 513], [1, 1, 1], nkv, hd, 16, seed=i)
        qkv = qkv_rows(3, nh, nkv, hd, i)
        out = torch.zeros(3, nh, hd, dtype=torch.float16, device=DEV)

        def step(c=c, qkv=qkv, out=out):
            q = ops.paged_kv_write(qkv, *c.args, n_heads=nh, cos=cos, sin=sin, **c.scales)
            ops.paged_attention(q, *c.args, out=out, **c.scales)

        step()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                step()
        graphs.append((gr, s, c, qkv, out, step))
    torch.cuda.synchronize()
    for kv, ql in shapes:
        want = []
        for gr, s, c, qkv, out, step in graphs:
            c.len_t.copy_(torch.tensor(kv, dtype=torch.int32))
            c.cu.copy_(torch.tensor([0] + list(np.cumsum(ql)), dtype=torch.int32))
            out.fill_(7.0)
            step()
            torch.cuda.synchronize()
            want.append((out.clone(), c.k.clone()))
            out.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(5):
            for gr, s, *_ in graphs:
                with torch.cuda.stream(s):
                    gr.replay()
        torch.cuda.synchronize()
        for (o, k), (gr, s, c, qkv, out, step) in zip(want, graphs):
            assert torch.equal(out, o) and torch.equal(c.k.view(torch.uint8), k.view(torch.uint8))
    assert faults() == 0


@pytest.mark.parametrize("ql", [1, 64])
def test_other_streams(ql):
    """Two streams at once, one given by argument; nothing is shared between the calls."""
    from atomflow_b200 import ops
    c = Cache("int8", [3000] * 2, [ql] * 2, 1, 128, 16)
    q, want = check_attention(c, 4, max_q=ql, tail=0)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(20):
        outs.append(ops.paged_attention(q, *c.args, max_q=ql, **c.scales, stream=s1))
        with torch.cuda.stream(s2):
            outs.append(ops.paged_attention(q, *c.args, max_q=ql, **c.scales))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("fmt", list(FMT))
def test_a_prompt_in_chunks_then_tokens(fmt):
    """As a serving loop runs them: a prompt written and attended chunk by chunk, then token by token, a second sequence
    beside it; the cache read back holds what was written, and every step's attention is that of the cache."""
    from atomflow_b200 import ops
    nh, nkv, hd, page = 6, 2, 128, 16
    cos, sin = rope_tables(256, hd)
    c = Cache(fmt, [200, 200], [0, 0], nkv, hd, page)
    total = [0, 0]
    for step, ql in enumerate([[100, 1], [37, 30], [1, 1], [1, 1], [2, 0]]):
        total = [a + b for a, b in zip(total, ql)]
        c.kv_len, c.q_len, c.T = total, ql, sum(ql)
        c.len_t.copy_(torch.tensor(total, dtype=torch.int32))
        c.cu.copy_(torch.tensor([0, ql[0], sum(ql)], dtype=torch.int32))
        qkv = qkv_rows(c.T, nh, nkv, hd, step)
        q = ops.paged_kv_write(qkv, *c.args, n_heads=nh, cos=cos, sin=sin, **c.scales)
        k, v = ops.paged_kv_read(*c.args, c.T, **c.scales)
        x = qkv.view(c.T, -1, hd)[:, nh + nkv:].float()
        # quantised: half a step of the code plus the value's FP16 rounding
        step_v = {"f16": 0.0, "fp8": 2.0 ** -4, "int8": 0.0}[fmt] * x.abs()
        if fmt != "f16":
            step_v = step_v + x.abs().amax(-1, keepdim=True) * ({"fp8": 2.0 ** -10 / 448, "int8": 0.5 / 127}[fmt] * (1 + 2.0 ** -10) + 2.0 ** -11)
        assert ((v.float() - x).abs() <= step_v).all()
        check_attention(c, nh, q=q, max_q=max(ql), max_kv=200)
    assert faults() == 0


def _with_bad_values(fmt, ql, where, ctx, nkv=2, hd=128, page=16, bad=(math.inf, -math.inf, math.nan)):
    """A cache whose V holds infinities and NaN at some positions of the last chunk, and the same without them."""
    n = ctx + ql
    c, clean = Cache(fmt, [n], [ql], nkv, hd, page, seed=7), Cache(fmt, [n], [ql], nkv, hd, page, seed=7)
    dims = torch.arange(0, hd, 37, device=DEV)
    for i, pos in enumerate(where):
        pg, slot = c.where(0, pos, 1)
        x = bad[i % len(bad)]
        if fmt == "f16":
            c.v[pg, slot, :, dims] = x
        elif fmt == "fp8":
            c.v.view(torch.uint8)[pg, slot, :, dims] = 0x7f          # the format has no infinity
        else:
            c.vs[pg, slot] = x                                       # the whole vector
        if fmt != "int8":
            c.k[pg, slot] = torch.full_like(c.k[pg, slot].float(), math.nan).to(c.k.dtype)
    return c, clean, dims


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("ql,ctx,hd", [(4, 300, 128), (4, 0, 64), (3, 5000, 128), (40, 100, 128), (200, 0, 64), (130, 9000, 128)])
def test_infinities_and_nan_reach_only_the_rows_that_see_them(fmt, ql, ctx, hd):
    """K and V of a chunk's later tokens are not finite: the earlier tokens' outputs do not change by a bit, the later
    ones' are not finite where V is not."""
    from atomflow_b200 import ops
    first = ctx + ql // 2
    c, clean, dims = _with_bad_values(fmt, ql, [first, ctx + ql - 1], ctx, hd=hd)
    q = torch.randn(ql, 4, hd, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0)).half()
    for kw in (dict(max_q=ql, max_kv=ctx + ql), dict(max_q=ql, max_kv=1)):
        got = ops.paged_attention(q, *c.args, **c.scales, **kw)
        ref = ops.paged_attention(q, *clean.args, **clean.scales, **kw)
        assert torch.equal(got[:ql // 2], ref[:ql // 2]) and torch.isfinite(ref).all()
        seen = got[ql // 2:].float()
        assert not torch.isfinite(seen if fmt == "int8" else seen[:, :, dims]).any()
        if fmt != "f16":
            assert seen[:, :, dims].isnan().any()
    assert faults() == 0


def test_an_infinity_in_v_gives_an_infinity():
    """Finite K: the rows that see +inf in V are +inf there, exact elsewhere, in both kernels."""
    from atomflow_b200 import ops
    for ql in (3, 100):
        c = Cache("f16", [300], [ql], 1, 128, 16, seed=2)
        q, good = check_attention(c, 2, max_q=ql, tail=0)
        pg, slot = c.where(0, 300 - ql // 2, 1)
        c.v[pg, slot, 0, 5] = math.inf
        out = ops.paged_attention(q, *c.args, max_q=ql)
        rows = ql - ql // 2
        assert torch.equal(out[:rows], good[:rows])
        assert (out[rows:, :, 5] == math.inf).all()
        assert torch.isfinite(out[rows:, :, 6:]).all()


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ql", [3, 300])
def test_scales_of_every_size(fmt, hd, ql):
    """Neighbouring positions whose scales differ by powers of ten, down to subnormal ones, over many tiles."""
    g = torch.Generator().manual_seed(hd + ql)
    ctx = 2300
    def values(low, high):
        x = torch.randn(ctx, 2, hd, generator=g)
        return x * 10.0 ** (torch.rand(ctx, 2, 1, generator=g) * (high - low) + low)
    c = Cache(fmt, [ctx], [ql], 2, hd, 16, k=[values(-5, 0.3)], v=[values(-5, 3)])
    assert (c.vs[c.where(0, 0, ctx)].float() < 2.0 ** -14).any()
    check_attention(c, 4)
    check_attention(c, 4, max_q=ql, max_kv=ctx)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_scales_that_are_not_finite(fmt, hd, which, bad):
    """Only the rows that see the position notice; the others are as with a scale of 1 there.  (K's scale multiplies
    the score: an infinite one makes it +inf, the row NaN, or -inf, the weight zero.)"""
    from atomflow_b200 import ops
    ctx, at = 700, 600
    for ql, first in ((300, 200), (16, 0), (2, 0)):   # from which row on it is seen
        c = Cache(fmt, [ctx], [ql], 2, hd, 16)
        pg, slot = (int(x) for x in c.where(0, at, 1))
        scale = c.ks if which == "k" else c.vs
        q = torch.randn(ql, 4, hd, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).half()
        scale[pg, slot] = 1.0
        want = ops.paged_attention(q, *c.args, **c.scales)
        dot = torch.einsum("thd,hd->th", q.double(), c.values(0, at, 1)[0][0].repeat_interleave(2, 0))
        scale[pg, slot] = bad
        got = ops.paged_attention(q, *c.args, **c.scales)
        assert faults() == 0
        assert torch.equal(got[:first], want[:first])
        got, dot = got[first:], dot[first:]
        if math.isnan(bad):
            assert got.isnan().all()
        elif which == "v":
            assert not got.isfinite().any()
        else:
            assert (dot.abs() > 2.0 ** -10).all()
            assert got[dot > 0].isnan().all() and got[dot < 0].isfinite().all()


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_mixed_batch_in_a_graph(fmt):
    """Both kernels of a mixed batch, overlapping, captured with the write and the read around them and replayed: as eager."""
    from atomflow_b200 import ops
    nh, nkv, hd = 8, 2, 128
    kv, ql = [700, 300, 5000, 64, 900, 33], [200, 1, 1, 64, 1, 3]
    cos, sin = rope_tables(5000, hd)
    c = Cache(fmt, kv, ql, nkv, hd, 16)
    qkv = qkv_rows(c.T, nh, nkv, hd, 5)

    def step():
        q = ops.paged_kv_write(qkv, *c.args, n_heads=nh, cos=cos, sin=sin, **c.scales)
        o = ops.paged_attention(q, *c.args, max_q=200, max_kv=5000, **c.scales)
        return (q, o) + tuple(ops.paged_kv_read(*c.args, c.T, **c.scales))

    eager = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs = step()
    for _ in range(3):
        for t in outs:
            t.fill_(5.0)
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, eager)) and faults() == 0
    check_attention(c, nh, q=eager[0], max_q=200, max_kv=5000)


def test_many_sequences_and_heads():
    """More sequences than a warp looks at in one step, more kv heads than a CTA has warps, both kernels."""
    kv = [1 + (37 * i) % 120 for i in range(150)]
    ql = [min(n, 30) if i % 11 == 0 else min(n, 1 + i % 3) for i, n in enumerate(kv)]
    c = Cache("int8", kv, ql, 3, 64, 8)
    check_attention(c, 6, max_q=30, max_kv=120)
    c = Cache("f16", [40] * 70, [1] * 70, 20, 64, 16)
    check_attention(c, 20, max_q=1)


@pytest.mark.parametrize("nh,nkv", [(64, 1), (200, 1)])
def test_large_groups(nh, nkv):
    """One kv head for many query heads: a single token's rows are a chunk's."""
    c = Cache("fp8", [300, 17], [1, 3], nkv, 128, 16)
    check_attention(c, nh, max_q=3, max_kv=300)


def test_without_a_workspace():
    """The C entry point with no workspace, or too small a one, gives the same result within the tolerance."""
    import ctypes

    from atomflow_b200 import lib
    from atomflow_b200._lib import PagedBatch, PagedKv
    c = Cache("f16", [40000, 9000], [1, 1], 1, 128, 64)
    q, want = check_attention(c, 4, max_q=1, max_kv=40000, tail=0)
    kv = PagedKv(0, c.k.shape[0], 64, 1, 128, c.k.data_ptr(), c.v.data_ptr(), c.k.stride(0), None, None, 0)
    b = PagedBatch(2, 2, c.table.shape[1], c.cu.data_ptr(), c.len_t.data_ptr(), c.table.data_ptr(), c.table.shape[1])
    L, R = lib(), ctypes.byref
    need = L.af_paged_attention_workspace_bytes(R(kv), R(b), 4, 1, 40000)
    assert need > 0
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device=DEV)     # any contents
    st = torch.cuda.current_stream().cuda_stream
    outs = []
    for ptr, n in ((None, 0), (ws.data_ptr(), need - 1), (ws.data_ptr(), need), (ws.data_ptr(), need)):
        out = torch.zeros_like(q)
        assert L.af_paged_attention(R(kv), R(b), q.data_ptr(), 4 * 128, 4, 128 ** -0.5, 1, 40000, out.data_ptr(), ptr, n, st) == 0
        outs.append(out)
    assert faults() == 0
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[3]) and torch.equal(outs[2], want)
    row = 0
    for i in range(2):
        ref, tol = attention_f64(c, q, 128 ** -0.5, i, row)
        assert ((outs[0][row:row + 1].double() - ref).abs() <= tol).all()
        row += 1


def test_refusals_of_the_library_reach_python():
    from atomflow_b200 import AtomflowError, ops
    c = Cache("f16", [16], [1], 1, 64, 16)
    q = torch.zeros(1, 2, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(AtomflowError, match="invalid"):
        ops.paged_attention(q, *c.args, scale=-1.0)
    with pytest.raises(AtomflowError, match="invalid"):
        ops.paged_attention(q, *c.args, out=q)                        # the output over the input
    big = torch.zeros(2, 16, 1, 96, dtype=torch.float16, device=DEV)
    with pytest.raises(AtomflowError, match="unsupported"):
        ops.paged_attention(torch.zeros(1, 2, 96, dtype=torch.float16, device=DEV), big, big, *c.args[2:])
    with pytest.raises(ValueError, match="pages' device"):
        ops.paged_attention(q.cpu(), *c.args)
    with pytest.raises(ValueError, match="one CUDA device"):
        ops.paged_attention(q, *c.args[:3], c.len_t.cpu(), c.cu)
    assert ops.paged_attention(q[:0], *c.args).shape == (0, 2, 64)    # nothing to do
    assert faults() == 0
