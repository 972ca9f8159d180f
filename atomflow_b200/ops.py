"""Host-side operators over the C ABI, for callers that hold torch CUDA tensors.

PyTorch here is plumbing (device memory, the current stream); all arithmetic
runs in libatomflow_b200.so.  Each op mirrors a reference launcher:

  w8a16_gemv  <- launch_w8a16_gemv   (include/ops/kernel.h:138-145)
  lm_head     <- engine.cu:494-513 cublasGemmEx + argmax launch (engine.cu:521)
  argmax      <- launch_argmax       (include/ops/kernel.h:155-159)

The paged_* ops have no reference launcher: a batch of sequences over a KV
cache in pages (FP16, FP8-E4M3 or INT8), described in include/atomflow_b200.h.
"""
import contextlib
import ctypes
import math

import torch

from ._lib import ArgmaxMode, KvFormat, PagedBatch, PagedKv, ScaleKind, WeightDtype, check, lib


def _stream(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


class Workspace:
    """Zero-initialised device scratch that grows on demand.  Kernels leave it
    zeroed again, so one Workspace serves every call issued on one stream."""

    def __init__(self, device=None, nbytes=1 << 20):
        self.device = torch.device(device or "cuda")
        self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)

    def get(self, nbytes):
        if self.buf.numel() < nbytes:
            torch.cuda.current_stream(self.device).synchronize()
            self.buf = torch.zeros(max(nbytes, 2 * self.buf.numel()), dtype=torch.uint8,
                                   device=self.device)
        return self.buf.data_ptr(), self.buf.numel()


_default_ws = {}


def default_workspace(device) -> Workspace:
    d = torch.device(device)
    key = d.index if d.index is not None else torch.cuda.current_device()
    if key not in _default_ws:
        _default_ws[key] = Workspace(torch.device("cuda", key))
    return _default_ws[key]


def _need(t, dtype, name):
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA {dtype} tensor")


def w8a16_gemv(x, w, scales=None, out=None, *, scale_kind="group", group_size=128,
               workspace=None, stream=None):
    """y[M, N] (fp16) = dequant(w[N, K] fp8) @ x[M, K] (fp16)^T, FP32 accumulation."""
    kind = {"group": ScaleKind.GROUP_F16, "row": ScaleKind.ROW_F32, "none": ScaleKind.NONE}[scale_kind]
    x2 = x.reshape(-1, x.shape[-1])
    M, K = x2.shape
    N = w.shape[0]
    _need(x2, torch.float16, "x")
    if w.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise ValueError("w must be float8_e4m3fn (or its uint8 bytes)")
    if out is None:
        out = torch.empty(M, N, dtype=torch.float16, device=x.device)
    _need(out, torch.float16, "out")
    L = lib()
    ws = workspace or default_workspace(x.device)
    need = L.af_w8a16_gemv_workspace_bytes(M, N, K, int(kind))
    ptr, nb = ws.get(need)
    check(L.af_w8a16_gemv(x2.data_ptr(), w.data_ptr(), scales.data_ptr() if scales is not None else None,
                          out.data_ptr(), M, N, K, group_size, int(kind), ptr, nb, _stream(stream)),
          "af_w8a16_gemv")
    return out


def lm_head(x, w, row_scale=None, logits=None, *, want_logits=True, want_argmax=True,
            mode="true", workspace=None, stream=None):
    """FP32 logits[V] = w[V, D] @ x[D]; optional fused greedy argmax (device int32[1])."""
    V, D = w.shape
    wdt = WeightDtype.F16 if w.dtype == torch.float16 else WeightDtype.FP8_E4M3
    if want_logits and logits is None:
        logits = torch.empty(V, dtype=torch.float32, device=x.device)
    idx = torch.empty(1, dtype=torch.int32, device=x.device) if want_argmax else None
    L = lib()
    ws = workspace or default_workspace(x.device)
    ptr, nb = ws.get(L.af_lm_head_workspace_bytes(V, D, int(wdt)))
    m = ArgmaxMode.TRUE if mode == "true" else ArgmaxMode.REF_COMPAT
    check(L.af_lm_head_gemv(x.data_ptr(), w.data_ptr(), int(wdt),
                            row_scale.data_ptr() if row_scale is not None else None,
                            logits.data_ptr() if want_logits else None, V, D,
                            idx.data_ptr() if idx is not None else None, int(m), ptr, nb,
                            _stream(stream)), "af_lm_head_gemv")
    return logits, idx


def argmax(logits, *, mode="true", out=None, workspace=None, stream=None):
    V = logits.shape[-1]
    _need(logits, torch.float32, "logits")
    if out is None:
        out = torch.empty(1, dtype=torch.int32, device=logits.device)
    L = lib()
    ws = workspace or default_workspace(logits.device)
    ptr, nb = ws.get(L.af_argmax_workspace_bytes(V))
    m = ArgmaxMode.TRUE if mode == "true" else ArgmaxMode.REF_COMPAT
    check(L.af_argmax_f32(logits.data_ptr(), V, out.data_ptr(), int(m), ptr, nb, _stream(stream)),
          "af_argmax_f32")
    return out


# ------------------------------------------------------------ paged KV cache
_KV_FORMATS = {torch.float16: KvFormat.F16, torch.float8_e4m3fn: KvFormat.FP8_E4M3, torch.int8: KvFormat.INT8}


def _paged(n_tokens, k_pages, v_pages, block_table, kv_len, cu_rows, k_scale, v_scale):
    """The C structures of a cache and a batch, checked (shapes, types, strides, one device)."""
    fmt = _KV_FORMATS.get(k_pages.dtype)
    if fmt is None or v_pages.dtype != k_pages.dtype:
        raise ValueError("k_pages and v_pages must both be float16, float8_e4m3fn or int8")
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride():
        raise ValueError("k_pages and v_pages must be [n_pages, page_size, n_kv_heads, head_dim], strided alike")
    n_pages, page, nkv, hd = k_pages.shape
    st = k_pages.stride()
    if st[1:] != (nkv * hd, hd, 1):
        raise ValueError("each page must be contiguous")
    page_stride = st[0] if n_pages > 1 else page * nkv * hd
    if (k_scale is None) != (fmt == 0) or (v_scale is None) != (fmt == 0):
        raise ValueError("8-bit pages need k_scale and v_scale, float16 pages take none")
    dev = k_pages.device
    ks = vs = None
    scale_stride = 0
    if k_scale is not None:
        want = (n_pages, page, nkv)
        if (k_scale.dtype != torch.float16 or v_scale.dtype != torch.float16 or k_scale.shape != want or
                v_scale.shape != want or k_scale.stride() != v_scale.stride() or
                k_scale.stride()[1:] != (nkv, 1)):
            raise ValueError("scales must be float16 [n_pages, page_size, n_kv_heads], each page contiguous, alike")
        if k_scale.device != dev or v_scale.device != dev:
            raise ValueError("every tensor must be on the pages' device")
        scale_stride = k_scale.stride(0) if n_pages > 1 else page * nkv
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    if (block_table.dtype != torch.int32 or block_table.dim() != 2 or kv_len.dtype != torch.int32 or
            cu_rows.dtype != torch.int32):
        raise ValueError("block_table must be int32 [n_seqs, max_pages], kv_len and the row offsets int32")
    n, width = block_table.shape
    if kv_len.shape != (n,) or cu_rows.shape != (n + 1,) or not kv_len.is_contiguous() or not cu_rows.is_contiguous():
        raise ValueError("kv_len must be [n_seqs], the row offsets [n_seqs + 1], contiguous")
    if width > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table's rows must be contiguous")
    if (not k_pages.is_cuda or v_pages.device != dev or block_table.device != dev or kv_len.device != dev or
            cu_rows.device != dev):
        raise ValueError("every tensor must be on one CUDA device")
    kv = PagedKv(fmt, n_pages, page, nkv, hd, k_pages.data_ptr(), v_pages.data_ptr(), page_stride, ks, vs,
                 scale_stride)
    batch = PagedBatch(n, n_tokens, width, cu_rows.data_ptr(), kv_len.data_ptr(), block_table.data_ptr(),
                       block_table.stride(0) if n > 1 else width)
    return kv, batch


def _need_rows(t, name, shape, device):
    """FP16 rows: the given shape, every row contiguous, rows any (aligned) distance apart."""
    if t.dtype != torch.float16 or t.device != device or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be a float16 tensor {list(shape)} on the pages' device")
    inner = 1
    for d in range(t.dim() - 1, 0, -1):
        if t.shape[d] != 1 and t.stride(d) != inner:
            raise ValueError(f"{name}'s rows must be contiguous")
        inner *= t.shape[d]
    return t.stride(0) if t.shape[0] > 1 else inner


@contextlib.contextmanager
def _on(device, stream):
    """The tensors' device and the stream of the call made current (so that what is allocated belongs to it)."""
    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield


def _launch(device, stream, call):
    """call(raw stream), with the tensors' device current."""
    if stream is None and device.index == torch.cuda.current_device():
        return call(torch.cuda.current_stream(device).cuda_stream)
    with _on(device, stream):
        return call(torch.cuda.current_stream(device).cuda_stream)


def paged_kv_write(qkv, k_pages, v_pages, block_table, kv_len, cu_rows, *, n_heads, cos=None, sin=None, k_scale=None,
                   v_scale=None, q_out=None, stream=None):
    """Stores a batch's new tokens in their pages (quantised, in 8-bit pages); in place.

    qkv fp16 [T, (n_heads + 2 * n_kv_heads) * head_dim], rows any distance apart.  With
    RoPE tables (fp32 [max_seq, head_dim / 2]) q and k are rotated at the tokens'
    positions; returns q [T, n_heads, head_dim]: rotated in q_out, or without tables
    qkv's own q."""
    nkv, hd = k_pages.shape[2:]
    T = qkv.shape[0]
    kv, batch = _paged(T, k_pages, v_pages, block_table, kv_len, cu_rows, k_scale, v_scale)
    dev = k_pages.device
    stride = _need_rows(qkv, "qkv", (T, (n_heads + 2 * nkv) * hd), dev)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is None:
        if q_out is not None:
            raise ValueError("q_out needs cos and sin: without them q is left in qkv")
    else:
        for t in (cos, sin):
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != hd // 2 or t.device != dev or \
                    t.shape != cos.shape or not t.is_contiguous():
                raise ValueError("cos and sin must be contiguous float32 [max_seq, head_dim / 2] on the pages' device")
        if q_out is not None and (_need_rows(q_out, "q_out", (T, n_heads, hd), dev) != n_heads * hd):
            raise ValueError("q_out must be contiguous")

    def call(s):
        q = q_out
        if q is None and cos is not None:
            q = torch.empty(T, n_heads, hd, dtype=torch.float16, device=dev)
        check(lib().af_paged_kv_write(ctypes.byref(kv), ctypes.byref(batch), qkv.data_ptr(), stride, n_heads,
                                      None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(),
                                      0 if cos is None else cos.shape[0], None if q is None else q.data_ptr(), s),
              "af_paged_kv_write")
        return qkv[:, :n_heads * hd].unflatten(1, (n_heads, hd)) if q is None else q

    return _launch(dev, stream, call)


def paged_kv_read(k_pages, v_pages, block_table, kv_len, cu_rows, n_rows, *, k_scale=None, v_scale=None, k_out=None,
                  v_out=None, stream=None):
    """The last cu_rows[b+1] - cu_rows[b] cached positions of each sequence as fp16 (k, v) [n_rows, n_kv_heads, head_dim]."""
    nkv, hd = k_pages.shape[2:]
    kv, batch = _paged(n_rows, k_pages, v_pages, block_table, kv_len, cu_rows, k_scale, v_scale)
    dev = k_pages.device
    for t in (k_out, v_out):
        if t is not None and _need_rows(t, "k_out and v_out", (n_rows, nkv, hd), dev) != nkv * hd:
            raise ValueError("k_out and v_out must be contiguous")

    def call(s):
        k = torch.empty(n_rows, nkv, hd, dtype=torch.float16, device=dev) if k_out is None else k_out
        v = torch.empty(n_rows, nkv, hd, dtype=torch.float16, device=dev) if v_out is None else v_out
        check(lib().af_paged_kv_read(ctypes.byref(kv), ctypes.byref(batch), k.data_ptr(), v.data_ptr(), s),
              "af_paged_kv_read")
        return k, v

    return _launch(dev, stream, call)


def paged_attention(q, k_pages, v_pages, block_table, kv_len, cu_rows, *, scale=None, k_scale=None, v_scale=None,
                    max_q=None, max_kv=None, out=None, stream=None):
    """Causal attention of a batch's new tokens over their cached positions, themselves included.

    q fp16 [T, n_heads, head_dim], tokens any distance apart; returns out, alike and
    contiguous.  scale: 1 / sqrt(head_dim) unless given.  max_q, max_kv: the host's bounds on
    any sequence's new tokens and cached positions, which choose the split of the work."""
    hd = k_pages.shape[3]
    if q.dim() != 3:
        raise ValueError("q must be [T, n_heads, head_dim]")
    T, nh = q.shape[:2]
    kv, batch = _paged(T, k_pages, v_pages, block_table, kv_len, cu_rows, k_scale, v_scale)
    dev = k_pages.device
    stride = _need_rows(q, "q", (T, nh, hd), dev)
    if out is not None and _need_rows(out, "out", (T, nh, hd), dev) != nh * hd:
        raise ValueError("out must be contiguous")
    if scale is None:
        scale = 1.0 / math.sqrt(hd)

    def call(s):
        o = torch.empty(T, nh, hd, dtype=torch.float16, device=dev) if out is None else out
        check(lib().af_paged_attention(ctypes.byref(kv), ctypes.byref(batch), q.data_ptr(), stride, nh, scale,
                                       max_q or 0, max_kv or 0, o.data_ptr(), s), "af_paged_attention")
        return o

    return _launch(dev, stream, call)
