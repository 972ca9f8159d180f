"""Attention over the paged KV cache with values that are not drawn from one normal distribution: queries and
keys that lean to one side, outlier channels, vectors of zeros, small values.  Caches, the 64-bit form and its
tolerance are those of test_paged_gpu.py."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_gpu import DEV, Cache, attention_f64, faults   # noqa: E402


def gen(seed):
    return torch.Generator().manual_seed(seed)


def compare(c, q, scale=None, extra=0.0, **kw):
    """Each output within attention_f64's tolerance plus `extra`."""
    from atomflow_b200 import ops
    got = ops.paged_attention(q, *c.args, scale=scale, **c.scales, **kw)
    assert faults() == 0
    row = 0
    for b, m in enumerate(c.q_len):
        want, tol = attention_f64(c, q, c.hd ** -0.5 if scale is None else scale, b, row)
        ratio = ((got[row:row + m].double() - want).abs() / (tol + extra)).nan_to_num(nan=9e9)
        assert float(ratio.max()) <= 1, (b, float(ratio.max()))
        row += m


# ---------------------------------------------------------------- one-sided values
# The score's tolerance is relative to sum |q_d k_d|: an operand format that adds a constant to every code would have
# partial sums far above it.
@pytest.mark.parametrize("fmt", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ql", [1, 4, 64])
def test_one_sided_queries_and_an_outlier_channel(fmt, hd, ql):
    """Keys of small whole numbers beside one channel of 127 that the query does not look at; the query's other
    elements are all near +20."""
    n = 700
    k = torch.randint(-1, 2, (n, 2, hd), generator=gen(1)).float()
    k[..., 5] = 127.0
    q = 20 + torch.randn(ql, 8, hd, generator=gen(2))
    q[..., 5] = 0.0
    c = Cache(fmt, [n], [ql], 2, hd, 16, k=[k])
    for scale in (0.01, 0.05):
        compare(c, q.half().to(DEV), scale=scale, max_q=ql, max_kv=n)


@pytest.mark.parametrize("fmt", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("mean,std", [(3, 1), (10, 5), (-20, 1)])
def test_queries_with_a_mean(fmt, hd, mean, std):
    c = Cache(fmt, [300, 41, 1000], [1, 2, 4], 2, hd, 16)
    q = (mean + std * torch.randn(7, 8, hd, generator=gen(3))).half().to(DEV)
    compare(c, q, max_q=4, max_kv=1000)
    compare(c, q, scale=0.02)


# ---------------------------------------------------------------- V of very different sizes
# P times the rest of V's scale is rounded to FP16: 2^-11 of itself, or, where it is subnormal, 2^-25, times a code and its
# power of two: at most max|v_j|, and for E4M3 scales below the smallest power (2^-15) at most 448 2^-14 (either kernel).
def tiny(c):
    return 2.0 ** -25 * 448 * 2.0 ** -14 * max(c.kv_len) if c.fmt == "fp8" else 0.0


def peaked(n, nkv, hd, top, seed):
    """Keys whose position `top` scores 8 above the others, which differ a little, for queries with 8 in element 0."""
    k = 0.3 * torch.randn(n, nkv, hd, generator=gen(seed))
    k[..., 0] = 0.0
    k[top, :, 0] = hd ** 0.5
    return k


def peaked_queries(ql, nh, hd, seed):
    q = torch.randn(ql, nh, hd, generator=gen(seed))
    q[..., 0] = 8.0
    return q.half().to(DEV)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ql", [1, 4, 64])
@pytest.mark.parametrize("std", [0.02, 0.005, 0.0005])
@pytest.mark.parametrize("sink", [True, False])
def test_zero_vectors_beside_small_values(fmt, hd, ql, std, sink):
    """V of ordinary small values with vectors of zeros among them, whose scale is 1; the position with the largest weight
    one of them, or not."""
    n, nkv = 2048, 2
    v = std * torch.randn(n, nkv, hd, generator=gen(4))
    v[7::50] = 0.0
    top = 57 if sink else 60
    c = Cache(fmt, [n], [ql], nkv, hd, 16, k=[peaked(n, nkv, hd, top, 5)], v=[v])
    assert (c.vs[c.where(0, 57, 1)] == 1).all() and (c.vs[c.where(0, 60, 1)] < 2.0 ** -10).all()
    q = peaked_queries(ql, 8, hd, 6)
    compare(c, q, extra=tiny(c), max_q=ql, max_kv=n)
    compare(c, q, extra=tiny(c))


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ql", [1, 64])
def test_an_outlier_vector_in_v(fmt, hd, ql):
    """One vector 2^12 times the others, at a score so low that it hardly counts: the others keep their bits."""
    n, nkv = 1000, 2
    v = 0.02 * torch.randn(n, nkv, hd, generator=gen(7))
    v[3::64] *= 4096.0
    k = peaked(n, nkv, hd, 500, 8)
    k[3::64, :, 0] = -2 * hd ** 0.5
    c = Cache(fmt, [n], [ql], nkv, hd, 16, k=[k], v=[v])
    q = peaked_queries(ql, 8, hd, 9)
    compare(c, q, extra=tiny(c), max_q=ql, max_kv=n)


# ---------------------------------------------------------------- scales above those that the write stores
def large_scales(fmt, ql, hd, n=1000, nkv=2):
    """A pool filled by the caller: V's scales up to FP16's largest, values beyond FP16 that average out."""
    c = Cache(fmt, [n], [ql], nkv, hd, 16, k=[0.1 * torch.randn(n, nkv, hd, generator=gen(10))])
    at = c.where(0, 0, n)
    e = torch.rand(n, nkv, generator=gen(11)) * 7 + 9                       # 2^9 .. 2^16
    c.vs[at] = (2.0 ** e).clamp(max=65504.0).half().to(DEV)
    c.vs[c.where(0, 500, 1)] = 65504.0
    if fmt == "int8":
        c.v[c.where(0, 17, 1)] = -128
    return c


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ql", [1, 4, 64])
def test_scales_above_the_stored_ones(fmt, hd, ql):
    """code * scale is not rounded to FP16: both kernels give the average, or an infinity where it is none of FP16."""
    from atomflow_b200 import ops
    c = large_scales(fmt, ql, hd)
    q = torch.randn(ql, 8, hd, generator=gen(12)).half().to(DEV)
    got = ops.paged_attention(q, *c.args, max_q=ql, max_kv=1000, **c.scales).double()
    want, tol = attention_f64(c, q, hd ** -0.5, 0, 0)
    assert faults() == 0 and not got.isnan().any()
    inside = want.abs() + tol < 65504
    assert inside.double().mean() > 0.05 and float(((got - want).abs() / tol)[inside].max()) <= 1
    outside = want.abs() - tol > 65520
    assert got[outside].isinf().all() and (got.sign() == want.sign())[outside].all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ql", [4, 64])
def test_nan_beside_values_beyond_fp16(hd, ql):
    """What is put back for the rows that see a NaN is the NaN alone, not finite values that are none of FP16."""
    from atomflow_b200 import ops
    c = large_scales("fp8", ql, hd)
    q = torch.randn(ql, 8, hd, generator=gen(13)).half().to(DEV)
    c.vs[c.where(0, 0, 1000)] = 1.0
    at = c.where(0, 1000 - ql // 2, ql // 2)                                # the last positions, masked for the first rows
    c.vs[at] = 1024.0
    c.v[at] = torch.full((ql // 2, 2, hd), 448.0, device=DEV).to(torch.float8_e4m3fn)
    clean = ops.paged_attention(q, *c.args, max_q=ql, max_kv=1000, **c.scales)
    c.v.view(torch.uint8)[c.where(0, 999, 1) + (slice(None), 3)] = 0x7f
    got = ops.paged_attention(q, *c.args, max_q=ql, max_kv=1000, **c.scales)
    assert faults() == 0 and torch.equal(got[:-1], clean[:-1]) and got[-1, :, 3].isnan().all()
    assert torch.equal(got[-1, :, :3], clean[-1, :, :3]) and torch.equal(got[-1, :, 4:], clean[-1, :, 4:])
