"""The paged KV cache without a GPU: the index arithmetic that the kernels share
(compiled for the host), and the refusals of the C entry points and the torch
ops, which return before any CUDA call."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
ROOT = Path(__file__).resolve().parents[1]
INT_MIN = -2 ** 31


# ------------------------------------------------------- index arithmetic
@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_index")
    (d / "t.cpp").write_text('''
#include "af_paged_index.h"
using namespace af;
extern "C" {
void seq(int s, int e, int kv, int n, int mp, int sh, int* out) {
    PagedSeq q = paged_seq_of(s, e, kv, n, mp, sh); out[0] = q.row0; out[1] = q.q; out[2] = q.kv; out[3] = q.bad;
}
int pos(int row0, int q, int kv, int t) { return paged_pos_of(PagedSeq{row0, q, kv, false}, t); }
int page_ok(int page, int n) { return paged_page_ok(page, n); }
int slot(int p, int sh) { return paged_slot_of(p, sh); }
long long table(int b, long long st, int p, int sh) { return paged_table_at(b, st, p, sh); }
long long vec(int page, long long pb, int slot, int nkv, int h, int vb) { return paged_vector_at(page, pb, slot, nkv, h, vb); }
long long scale(int page, long long st, int slot, int nkv, int h) { return paged_scale_at(page, st, slot, nkv, h); }
}''')
    so = d / "t.so"
    subprocess.run(["g++", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-std=c++17", "-I",
                    str(ROOT / "atomflow_b200" / "csrc"), "-o", str(so), str(d / "t.cpp"), "-lubsan"], check=True)
    h = ctypes.CDLL(str(so))
    for f in ("table", "vec", "scale"):
        getattr(h, f).restype = ctypes.c_longlong
    return h


def _seq(h, *args):
    out = (ctypes.c_int * 4)()
    h.seq(*args, out)
    return tuple(out)


def test_sequences_outside_the_buffers_have_no_rows(index):
    assert _seq(index, 3, 7, 40, 10, 4, 4) == (3, 4, 40, 0)
    assert _seq(index, 3, 3, 0, 10, 0, 4) == (3, 0, 0, 0)            # empty
    assert _seq(index, 0, 10, 64, 10, 4, 4) == (0, 10, 64, 0)        # exactly full table
    for bad in [(-1, 4, 8, 10, 4, 4), (5, 4, 8, 10, 4, 4), (0, 11, 16, 10, 4, 4), (0, 4, -1, 10, 4, 4),
                (0, 4, 65, 10, 4, 4), (0, 4, 1, 10, 0, 4), (INT_MIN, 4, 8, 10, 4, 4), (2 ** 31 - 1, INT_MIN, 0, 10, 4, 4),
                (0, 2 ** 31 - 1, 4, 10, 4, 4)]:
        assert _seq(index, *bad) == (0, 0, 0, 1), bad
    # a table as wide as an int can say: the product does not overflow
    assert _seq(index, 0, 1, 2 ** 30, 1, 2 ** 31 - 1, 8) == (0, 1, 2 ** 30, 0)
    assert _seq(index, 0, 1, 2 ** 30 + 1, 1, 2 ** 31 - 1, 8) == (0, 0, 0, 1)


def test_positions_of_rows(index):
    assert [index.pos(3, 4, 40, t) for t in (2, 3, 6, 7)] == [INT_MIN, 36, 39, INT_MIN]
    assert [index.pos(0, 5, 2, t) for t in range(5)] == [-3, -2, -1, 0, 1]    # longer than its cache
    assert index.pos(0, 0, 9, 0) == INT_MIN
    assert index.pos(0, 1, 2 ** 31 - 1, 0) == 2 ** 31 - 2


def test_bad_pages_are_refused(index):
    assert [index.page_ok(p, 7) for p in (-1, 0, 6, 7, INT_MIN, 2 ** 31 - 1)] == [0, 1, 1, 0, 0, 0]
    assert index.page_ok(0, 0) == 0


def test_offsets_pass_32_bits(index):
    rng = random.Random(0)
    L = ctypes.c_longlong
    for _ in range(2000):
        sh = rng.randint(3, 8)
        pos, b = rng.randrange(2 ** 31 - 1), rng.randrange(2 ** 20)
        st = rng.choice([0, 1, 300, 2 ** 33])
        assert index.slot(pos, sh) == pos % 2 ** sh
        assert index.table(b, L(st), pos, sh) == b * st + pos // 2 ** sh
        page, nkv = rng.randrange(2 ** 31 - 1), rng.randint(1, 1024)
        slot, head = rng.randrange(2 ** sh), rng.randrange(nkv)
        pb = rng.choice([2 ** sh * nkv * 256, 2 ** 31 + 16])
        assert index.vec(page, L(pb), slot, nkv, head, 256) == page * pb + (slot * nkv + head) * 256
        assert index.scale(page, L(pb), slot, nkv, head) == page * pb + slot * nkv + head


# ------------------------------------------------------- refusals, C ABI
def _c(**over):
    from atomflow_b200._lib import PagedBatch, PagedKv
    kv = dict(format=0, n_pages=4, page_size=16, n_kv_heads=2, head_dim=128, k=4096, v=4096, page_stride=16 * 256,
              k_scale=None, v_scale=None, scale_stride=0)
    b = dict(n_seqs=1, n_tokens=1, max_pages=2, cu_rows=4096, kv_len=4096, block_table=4096, table_stride=2)
    for k, v in over.items():
        (kv if k in kv else b)[k] = v
    return PagedKv(**kv), PagedBatch(**b)


def _calls(kv, b):
    from atomflow_b200._lib import lib
    L, R = lib(), ctypes.byref
    return [L.af_paged_kv_write(R(kv), R(b), 4096, 8 * 128, 4, None, None, 0, None, None),
            L.af_paged_kv_read(R(kv), R(b), 4096, 4096, None),
            L.af_paged_attention(R(kv), R(b), 4096, 4 * 128, 4, 0.1, 0, 0, 4096, None, 0, None)]


@pytest.mark.parametrize("over,status", [
    (dict(format=3), 1), (dict(format=-1), 1), (dict(head_dim=96), 2), (dict(head_dim=256), 2), (dict(n_pages=-1), 1),
    (dict(page_size=4), 2), (dict(page_size=24), 2), (dict(page_size=512), 2), (dict(n_kv_heads=0), 1),
    (dict(k=None), 1), (dict(v=None), 1), (dict(k=4104), 1), (dict(page_stride=16 * 256 - 8), 1),
    (dict(page_stride=16 * 256 + 4), 1), (dict(k_scale=4096, v_scale=4096), 1),
    (dict(format=1), 1), (dict(format=1, k_scale=4096, v_scale=4096, scale_stride=31), 1),
    (dict(format=2, k_scale=4096, scale_stride=32), 1), (dict(format=2, k_scale=4097, v_scale=4096, scale_stride=32), 1),
    (dict(format=2, k_scale=4096, v_scale=4096, scale_stride=32, page_stride=16 * 256 + 8), 1),
    (dict(n_seqs=-1), 1), (dict(n_tokens=-1), 1), (dict(max_pages=-1), 1), (dict(table_stride=1), 1),
    (dict(cu_rows=None), 1), (dict(kv_len=None), 1), (dict(block_table=None), 1), (dict(kv_len=4098), 1),
    (dict(n_kv_heads=1025, page_stride=16 * 1025 * 128), 1)])
def test_bad_caches_and_batches_are_refused(over, status):
    assert _calls(*_c(**over)) == [status] * 3


def test_null_structures_and_empty_batches():
    from atomflow_b200._lib import lib
    L = lib()
    kv, b = _c()
    assert L.af_paged_kv_read(None, ctypes.byref(b), 4096, 4096, None) == 1
    assert L.af_paged_kv_read(ctypes.byref(kv), None, 4096, 4096, None) == 1
    assert _calls(*_c(n_seqs=0)) == [0, 0, 0]
    assert _calls(*_c(n_tokens=0, k=None, v=None, cu_rows=None)) == [0, 0, 0]


def test_bad_rows_are_refused():
    from atomflow_b200._lib import lib
    L, R = lib(), ctypes.byref
    kv, b = _c()
    far = 1 << 20

    def write(qkv=4096, stride=8 * 128, heads=4, cos=None, sin=None, max_seq=0, q=None):
        return L.af_paged_kv_write(R(kv), R(b), qkv, stride, heads, cos, sin, max_seq, q, None)

    def attend(q=4096, stride=4 * 128, heads=4, scale=0.1, rows=0, kvb=0, out=1 << 20, ws=None):
        return L.af_paged_attention(R(kv), R(b), q, stride, heads, scale, rows, kvb, out, ws, 0, None)

    assert write(qkv=None) == write(qkv=4104) == write(stride=8 * 128 - 8) == write(stride=8 * 128 + 4) == 1
    assert write(heads=-1) == write(cos=4096, q=far, max_seq=8) == write(cos=4096, sin=4096, q=far) == 1
    assert write(cos=4096, sin=4096, max_seq=8) == 1                        # no q_out
    assert write(cos=4104, sin=4096, max_seq=8, q=far) == 1
    # outputs over inputs, or over each other
    for q in (4096, 4096 + 2 * 8 * 128 - 16, 4096 - 2 * 4 * 128 + 16):
        assert write(cos=4096, sin=4096, max_seq=8, q=q) == 1
    for out in (4096, 4096 + 2 * 4 * 128 - 16, 4096 - 2 * 4 * 128 + 16):
        assert attend(out=out) == 1
    assert L.af_paged_kv_read(R(kv), R(b), 4096, 4096 + 2 * 2 * 128 - 16, None) == 1
    assert attend(q=None) == attend(out=None) == attend(q=4104) == attend(out=4104) == 1
    assert attend(stride=4 * 128 - 8) == attend(stride=4 * 128 + 4) == attend(heads=3) == attend(heads=0) == 1
    assert attend(rows=-1) == attend(kvb=-1) == attend(ws=4104) == 1
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert attend(scale=bad) == 1
    assert L.af_paged_kv_read(R(kv), R(b), None, 4096, None) == L.af_paged_kv_read(R(kv), R(b), 4096, 4104, None) == 1


# ------------------------------------------------------- refusals, torch ops
def _t(fmt=torch.float16, pages=4, page=16, nkv=2, hd=128, n=1, width=2, T=1, nh=4):
    t = dict(k_pages=torch.zeros(pages, page, nkv, hd).to(fmt), v_pages=torch.zeros(pages, page, nkv, hd).to(fmt),
             block_table=torch.zeros(n, width, dtype=torch.int32), kv_len=torch.ones(n, dtype=torch.int32),
             cu_rows=torch.arange(n + 1, dtype=torch.int32))
    s = dict(k_scale=None, v_scale=None)
    if fmt != torch.float16:
        s = dict(k_scale=torch.ones(pages, page, nkv, dtype=torch.float16), v_scale=torch.ones(pages, page, nkv, dtype=torch.float16))
    return t, s, torch.zeros(T, nh, hd, dtype=torch.float16)


@pytest.mark.parametrize("change,text", [
    (dict(k_pages=torch.zeros(4, 16, 2, 128)), "float16, float8"),
    (dict(v_pages=torch.zeros(4, 16, 2, 64, dtype=torch.float16)), "strided alike"),
    (dict(k_pages=torch.zeros(4, 16, 256, dtype=torch.float16), v_pages=torch.zeros(4, 16, 256, dtype=torch.float16)), "must be"),
    (dict(k_pages=torch.zeros(4, 2, 16, 128, dtype=torch.float16).transpose(1, 2),
          v_pages=torch.zeros(4, 2, 16, 128, dtype=torch.float16).transpose(1, 2)), "contiguous"),
    (dict(block_table=torch.zeros(1, 2, dtype=torch.int64)), "int32"), (dict(block_table=torch.zeros(2, dtype=torch.int32)), "int32"),
    (dict(kv_len=torch.ones(2, dtype=torch.int32)), "kv_len"), (dict(cu_rows=torch.zeros(3, dtype=torch.int32)), "offsets"),
    (dict(kv_len=torch.ones(1, dtype=torch.int64)), "int32"),
    (dict(block_table=torch.zeros(2, 1, dtype=torch.int32).t()), None),          # one row: any stride is refused or fine
    (dict(), "CUDA device")])
def test_ops_refuse_bad_tensors(change, text):
    from atomflow_b200 import ops
    t, s, q = _t()
    t.update(change)
    with pytest.raises(ValueError, match=text):
        ops.paged_attention(q, **t, **s)
    with pytest.raises(ValueError, match=text):
        ops.paged_kv_read(**t, n_rows=1, **s)
    with pytest.raises(ValueError, match=text):
        ops.paged_kv_write(torch.zeros(1, 8 * t["k_pages"].shape[-1], dtype=torch.float16), n_heads=4, **t, **s)


def test_ops_refuse_scales_that_do_not_fit_the_format():
    from atomflow_b200 import ops
    t, _, q = _t()
    one = torch.ones(4, 16, 2, dtype=torch.float16)
    with pytest.raises(ValueError, match="take no scales"):
        ops.paged_attention(q, **t, k_scale=one, v_scale=one)
    t8, s8, _ = _t(torch.int8)
    for bad in (dict(k_scale=None), dict(v_scale=None), dict(k_scale=one.float()), dict(v_scale=one[:3]),
                dict(k_scale=one.transpose(1, 2).contiguous().transpose(1, 2), v_scale=one)):
        with pytest.raises(ValueError, match="scale"):
            ops.paged_attention(q, **t8, **{**s8, **bad})
    with pytest.raises(ValueError, match="n_heads"):
        ops.paged_attention(q[0], **t8, **s8)


def test_ops_refuse_what_needs_a_gradient():
    from atomflow_b200 import ops
    t, s, q = _t()
    with pytest.raises(ValueError, match="no gradient"):
        ops.paged_attention(q.requires_grad_(), **t, **s)
    with pytest.raises(ValueError, match="no gradient"):
        ops.paged_kv_write(torch.zeros(1, 1024, dtype=torch.float16, requires_grad=True), n_heads=4, **t, **s)
    for name in ("k_pages", "v_pages"):
        bad = {**t, name: t[name].clone().requires_grad_()}
        with pytest.raises(ValueError, match="no gradient"):
            ops.paged_attention(q.detach(), **bad, **s)
        with pytest.raises(ValueError, match="no gradient"):
            ops.paged_kv_read(**bad, n_rows=1, **s)


def test_ops_refuse_what_is_no_tensor_or_number():
    from atomflow_b200 import ops
    t, s, q = _t()
    with pytest.raises(TypeError, match="q must be a tensor"):
        ops.paged_attention([1.0], **t, **s)
    with pytest.raises(TypeError):
        ops.paged_kv_read(**t, n_rows=1.5, **s)
    with pytest.raises(TypeError, match="cos must be a tensor"):
        ops.paged_kv_write(torch.zeros(1, 1024, dtype=torch.float16), n_heads=4, cos=3, sin=4, **t, **s)


def test_structures_match_the_header():
    from atomflow_b200._lib import PagedBatch, PagedKv
    assert ctypes.sizeof(PagedKv) == 72 and PagedKv.k.offset == 24 and PagedKv.scale_stride.offset == 64
    assert ctypes.sizeof(PagedBatch) == 48 and PagedBatch.cu_rows.offset == 16 and PagedBatch.table_stride.offset == 40
