"""The paged operators have no gradient, and say so: what asks for one is refused before anything else (no GPU needed)."""
import pytest

torch = pytest.importorskip("torch")
import torch.autograd.forward_ad as fwAD   # noqa: E402

from test_paged import _t   # noqa: E402


def tensors():
    t, _, q = _t(torch.int8)
    s = {name: torch.ones(4, 16, 2, dtype=torch.float16) for name in ("k_scale", "v_scale")}
    return t, s, q


def calls(t, s, q, qkv, **write):
    """The three operators on these tensors."""
    from atomflow_b200 import ops
    yield lambda: ops.paged_attention(q, **t, **s)
    yield lambda: ops.paged_kv_read(**t, n_rows=1, **s)
    yield lambda: ops.paged_kv_write(qkv, n_heads=4, **t, **s, **write)


def test_tangents_are_refused():
    """Dual tensors of forward-mode differentiation, under no_grad too: it does not turn that mode off."""
    f16, _, q = _t()
    t, s, _ = tensors()
    qkv = torch.zeros(1, 1024, dtype=torch.float16)
    with fwAD.dual_level():
        dual = lambda x: fwAD.make_dual(x, torch.ones_like(x))
        attend, _, write = calls(f16, {}, dual(q), dual(qkv))
        bad = [attend, write]
        for name in ("k_pages", "v_pages"):
            bad += list(calls({**f16, name: dual(f16[name])}, {}, q, qkv))
        for name in ("k_scale", "v_scale"):
            bad += list(calls(t, {**s, name: dual(s[name])}, q, qkv))
        for call in bad:
            with pytest.raises(ValueError, match="no gradient.*dual"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="no gradient.*dual"):
                call()
        for call in calls(f16, {}, q, qkv):   # none among the arguments: the next check's refusal
            with pytest.raises(ValueError, match="CUDA device"):
                call()


def test_outputs_and_tables_that_require_a_gradient_are_refused():
    from atomflow_b200 import ops
    t, _, q = _t()
    qkv, like = torch.zeros(1, 1024, dtype=torch.float16), torch.zeros(1, 2, 128, dtype=torch.float16)
    tab = torch.zeros(8, 64)
    grad = lambda x: x.clone().requires_grad_()
    bad = [lambda: ops.paged_attention(q, **t, out=grad(q)),
           lambda: ops.paged_kv_read(**t, n_rows=1, k_out=grad(like)),
           lambda: ops.paged_kv_read(**t, n_rows=1, v_out=grad(like)),
           lambda: ops.paged_kv_write(qkv, **t, n_heads=4, cos=grad(tab), sin=tab),
           lambda: ops.paged_kv_write(qkv, **t, n_heads=4, cos=tab, sin=grad(tab)),
           lambda: ops.paged_kv_write(qkv, **t, n_heads=4, cos=tab, sin=tab, q_out=grad(q))]
    for call in bad:
        with pytest.raises(ValueError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):   # there it is the caller's wish
            call()
