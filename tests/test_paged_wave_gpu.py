"""Attention of few rows where the work is cut into one wave of CTAs: long bounds, many sequences and heads.

The cut follows the host's bound on the cached positions, not the lengths, so the caches here are short and the bound (and
the table) is wide: MAX_KV is past what clusters of the largest size take.  `wave` says how many CTAs the plan has."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_gpu import DEV, FMT, Cache, attention_f64, faults, qkv_rows, rope_tables   # noqa: E402

MAX_KV = 8 * 2560 + 100


def widen(c, positions=MAX_KV):
    """The cache's table with room for `positions`, the new entries no pages."""
    width = -(-positions // c.page)
    t = torch.full((c.table.shape[0], width), -9, dtype=torch.int32, device=DEV)
    t[:, :c.table.shape[1]] = c.table
    c.table = t
    return c


def wave(c, nh, max_q, max_kv=MAX_KV):
    """Whether the plan for these bounds has CTAs of four warps (False) or one CTA per SM (True); fails where it is no wave."""
    from atomflow_b200 import lib
    from atomflow_b200._lib import PagedBatch, PagedKv
    fmt = list(FMT).index(c.fmt)
    scale = [None, None, 0] if fmt == 0 else [c.ks.data_ptr(), c.vs.data_ptr(), c.ks.stride(0)]
    kv = PagedKv(fmt, c.k.shape[0], c.page, c.nkv, c.hd, c.k.data_ptr(), c.v.data_ptr(), c.k.stride(0), *scale)
    b = PagedBatch(len(c.kv_len), c.T, c.table.shape[1], c.cu.data_ptr(), c.len_t.data_ptr(), c.table.data_ptr(),
                   c.table.shape[1])
    need = lib().af_paged_attention_workspace_bytes(ctypes.byref(kv), ctypes.byref(b), nh, max_q, max_kv)
    rows = 8 if max_q * (nh // c.nkv) <= 8 else 16
    ctas, rest = divmod(need, 2 * rows * (c.hd * 4 + 8) + 16)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert ctas > 0 and rest == 0 and ctas % sms == 0
    return ctas == sms


def check(c, nh, big, max_q, skip=(), fault=0, seed=1):
    """Every sequence against the 64-bit form but those of `skip`, which are left as they were; the same bits again."""
    from atomflow_b200 import ops
    assert wave(c, nh, max_q) == big
    q = torch.randn(c.T + 2, nh, c.hd, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).half()
    runs = []
    for _ in range(2):
        out = torch.full_like(q, 77.0)
        ops.paged_attention(q, *c.args, out=out, max_q=max_q, max_kv=MAX_KV, **c.scales)
        assert faults() == fault
        runs.append(out)
    assert torch.equal(*(r.view(torch.int16) for r in runs))
    out, row = runs[0], 0
    for b, m in enumerate(c.q_len):
        got = out[row:row + m]
        if b in skip:
            assert (got == 77.0).all(), b
        elif m:
            want, tol = attention_f64(c, q, c.hd ** -0.5, b, row)
            ratio = ((got.double() - want).abs() / tol.clamp(min=1e-30)).nan_to_num(nan=9e9)
            assert float(ratio.max()) <= 1, (b, float(ratio.max()))
        row += m
    assert (out[row:] == 77.0).all()


def ragged(n, top, seed):
    """Lengths from none to `top`, those of a tile's border among them."""
    g = torch.Generator().manual_seed(seed)
    kv = [int(top ** float(x)) for x in torch.rand(n, generator=g)]
    for i, x in enumerate((0, 1, 15, 16, 17, top, 127, 128)):
        kv[(5 * i + 2) % n] = x
    return kv


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,nkv,nh,ql", [(70, 2, 2, 1), (45, 3, 9, 1), (40, 2, 16, 2), (40, 2, 8, 4), (41, 1, 5, 3)])
def test_ragged_batches(fmt, hd, n, nkv, nh, ql):
    """One and sixteen rows per kv head; CTAs go on from head to head and over the sequences; more sequences than a warp
    looks at in one step."""
    kv = ragged(n, 1500, n)
    c = widen(Cache(fmt, kv, [min(ql, 1 + b % ql) if ql > 1 else 1 for b in range(n)], nkv, hd, 16, seed=n))
    check(c, nh, False, ql)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,nkv,nh,ql", [(3, 8, 8, 1), (4, 3, 24, 2), (1, 1, 4, 4), (9, 4, 8, 1)])
def test_few_items(fmt, hd, n, nkv, nh, ql):
    """One CTA per SM with all its warps, items cut into pieces at any place."""
    kv = [3000, 17, 900, 0, 5, 2100, 64, 300, 1][:n]
    c = widen(Cache(fmt, kv, [ql] * n, nkv, hd, 32, seed=3))
    check(c, nh, True, ql)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("n,nkv,nh,ql,kv,big", [(6, 8, 8, 1, 2000, False), (50, 2, 8, 4, 700, False), (4, 8, 32, 1, 2500, True),
                                                (5, 2, 16, 2, 4001, True), (37, 4, 4, 1, 16, False), (60, 8, 8, 1, 130, False)])
def test_equal_lengths(fmt, n, nkv, nh, ql, kv, big):
    """All sequences of one length: every item is cut at its own borders, or, with more items than CTAs, evenly."""
    c = widen(Cache(fmt, [kv] * n, [ql] * n, nkv, 128, 16, seed=4))
    check(c, nh, big, ql)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("nkv,nh,ql", [(2, 2, 1), (2, 16, 2)])
def test_sequences_that_are_not_ours_lie_between(fmt, nkv, nh, ql):
    """Empty ones, ones whose length their table cannot hold, ones of more rows than the bound says: those are left as
    they were, on both sides of a CTA's border, at the start and at the end."""
    n = 48
    kv, q = ragged(n, 1000, 9), [ql] * n
    empty, many = {0, 7, 8, 33, 40}, {3, 20, 21, 46}
    for b in empty:
        q[b] = 0
    for b in many:
        q[b] = 30
    c = widen(Cache(fmt, kv, q, nkv, 128, 16, seed=5))
    far = {1, 12, 31, 32, 47}
    for b in far:
        c.len_t[b] = 10 ** 6
    check(c, nh, False, ql, skip=many | far, fault=16)


@pytest.mark.parametrize("fmt", list(FMT))
def test_behind_the_chunks_in_a_graph(fmt):
    """Chunks by the one kernel, the others by a wave that begins beside it, with the write before and the read after
    them, captured and replayed: as eager, and right."""
    from atomflow_b200 import ops
    nh, nkv, hd, n = 8, 2, 128, 45
    kv = [max(x, 1) for x in ragged(n, 1200, 2)]
    ql = [1] * n
    for b, m in ((0, 200), (5, 40), (20, 513), (44, 33)):
        ql[b], kv[b] = m, max(kv[b], m)
    c = widen(Cache(fmt, kv, ql, nkv, hd, 16, seed=6))
    assert not wave(c, nh, 513)
    cos, sin = rope_tables(1300, hd)
    qkv = qkv_rows(c.T, nh, nkv, hd, 5)

    def step():
        q = ops.paged_kv_write(qkv, *c.args, n_heads=nh, cos=cos, sin=sin, **c.scales)
        o = ops.paged_attention(q, *c.args, max_q=513, max_kv=MAX_KV, **c.scales)
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
    row = 0
    for b, m in enumerate(ql):
        want, tol = attention_f64(c, eager[0], hd ** -0.5, b, row)
        assert ((eager[1][row:row + m].double() - want).abs() <= tol).all(), b
        row += m


@pytest.mark.parametrize("fmt", ["f16", "fp8"])
def test_infinities_and_nan_behind_a_row(fmt):
    """K and V of the drafts' last tokens are not finite, in every sequence of a wave: the earlier tokens do not notice."""
    from atomflow_b200 import ops
    n, nkv, ql = 40, 2, 4
    kv = [max(x, ql) for x in ragged(n, 900, 11)]
    make = lambda: widen(Cache(fmt, kv, [ql] * n, nkv, 128, 8, seed=8))
    c, clean = make(), make()
    assert not wave(c, 8, ql)
    for b in range(n):
        pg, slot = c.where(b, kv[b] - 2, 2)
        if fmt == "f16":
            c.v[pg, slot, :, ::37] = math.inf
            c.k[pg, slot] = math.nan
        else:
            c.v.view(torch.uint8)[pg, slot, :, ::37] = 0x7f
            c.k.view(torch.uint8)[pg, slot] = 0x7f
    q = torch.randn(c.T, 8, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).half()
    got, ref = (ops.paged_attention(q, *x.args, max_q=ql, max_kv=MAX_KV, **x.scales).view(n, ql, 8, 128) for x in (c, clean))
    assert faults() == 0 and torch.isfinite(ref).all()
    assert torch.equal(got[:, :2], ref[:, :2]) and not torch.isfinite(got[:, 2:, :, ::37]).any()
