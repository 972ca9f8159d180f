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
