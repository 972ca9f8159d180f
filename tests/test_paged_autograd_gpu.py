"""What the paged operators write in place, autograd knows of."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_gpu import Cache, faults, qkv_rows, rope_tables   # noqa: E402


@pytest.mark.parametrize("fmt", ["f16", "int8"])
def test_tensors_written_in_place_have_a_new_version(fmt):
    from atomflow_b200 import ops
    nh, nkv, hd = 4, 2, 64
    c = Cache(fmt, [20, 9], [3, 1], nkv, hd, 16)
    cos, sin = rope_tables(32, hd)
    qkv = qkv_rows(4, nh, nkv, hd, 0)
    new = lambda *shape: torch.empty(*shape, dtype=torch.float16, device="cuda")
    q, k, v, out = new(4, nh, hd), new(4, nkv, hd), new(4, nkv, hd), new(4, nh, hd)
    pools = [t for t in (c.k, c.v, c.ks, c.vs) if t is not None]

    def versions(*ts):
        return [t._version for t in ts]

    read_only = [qkv, cos, sin, c.table, c.len_t, c.cu]
    before, kept = versions(*pools, q), versions(*read_only)
    ops.paged_kv_write(qkv, *c.args, n_heads=nh, cos=cos, sin=sin, q_out=q, **c.scales)
    assert all(a < b for a, b in zip(before, versions(*pools, q)))
    before, kept = versions(k, v, out), kept + versions(*pools, q)
    ops.paged_kv_read(*c.args, 4, k_out=k, v_out=v, **c.scales)
    ops.paged_attention(q, *c.args, out=out, **c.scales)
    assert all(a < b for a, b in zip(before, versions(k, v, out)))
    assert versions(*read_only, *pools, q) == kept and faults() == 0


def test_a_backward_pass_over_a_cache_written_since_is_refused():
    from atomflow_b200 import ops
    c = Cache("f16", [20], [3], 2, 64, 16)
    w = torch.ones(64, device="cuda", dtype=torch.float16, requires_grad=True)
    y = (c.k * w).nan_to_num().sum()                    # saves the pages
    ops.paged_kv_write(qkv_rows(3, 0, 2, 64, 1), *c.args, n_heads=0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_tensors_of_inference_mode():
    from atomflow_b200 import ops
    with torch.inference_mode():
        c = Cache("int8", [20], [3], 2, 64, 16)
        out = torch.empty(3, 4, 64, dtype=torch.float16, device="cuda")
        qkv = qkv_rows(3, 4, 2, 64, 1)
    for mode in (torch.inference_mode(), torch.no_grad(), torch.enable_grad()):
        with mode:
            q = ops.paged_kv_write(qkv, *c.args, n_heads=4, **c.scales)
            assert ops.paged_attention(q, *c.args, out=out, **c.scales) is out
    assert faults() == 0
