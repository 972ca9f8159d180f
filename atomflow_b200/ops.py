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

import torch

from ._lib import ArgmaxMode, PagedBatch, PagedKv, ScaleKind, WeightDtype, check, lib


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
_KV_FORMATS = {torch.float16: 0, torch.float8_e4m3fn: 1, torch.int8: 2}   # _lib.KvFormat
_F16, _F32, _I32 = torch.float16, torch.float32, torch.int32


def _paged(n_tokens, k_pages, v_pages, block_table, kv_len, cu_rows, k_scale, v_scale):
    """The C structures of a cache and a batch, checked (shapes, types, strides, one device), and the device's index.

    A decode step calls this for every layer: each attribute of a tensor is read once."""
    fmt = _KV_FORMATS.get(k_pages.dtype)
    shape, st = k_pages.shape, k_pages.stride()
    if fmt is None or v_pages.dtype is not k_pages.dtype:
        raise ValueError("k_pages and v_pages must both be float16, float8_e4m3fn or int8")
    if len(shape) != 4 or v_pages.shape != shape or v_pages.stride() != st:
        raise ValueError("k_pages and v_pages must be [n_pages, page_size, n_kv_heads, head_dim], strided alike")
    n_pages, page, nkv, hd = shape
    row = nkv * hd
    if st[3] != 1 or st[2] != hd or st[1] != row:
        raise ValueError("each page must be contiguous")
    dev = k_pages.get_device()
    ks = vs = None
    scale_stride = 0
    if k_scale is None or v_scale is None or fmt == 0:
        if fmt != 0:
            raise ValueError("8-bit pages need k_scale and v_scale")
        if k_scale is not None or v_scale is not None:
            raise ValueError("float16 pages take no scales")
    else:
        sst = k_scale.stride()
        if (k_scale.dtype is not _F16 or v_scale.dtype is not _F16 or k_scale.shape != shape[:3] or
                v_scale.shape != shape[:3] or v_scale.stride() != sst or sst[2] != 1 or sst[1] != nkv):
            raise ValueError("scales must be float16 [n_pages, page_size, n_kv_heads], each page contiguous, alike")
        if k_scale.get_device() != dev or v_scale.get_device() != dev:
            raise ValueError("every tensor must be on one CUDA device")
        scale_stride = sst[0] if n_pages > 1 else page * nkv
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    table_shape = block_table.shape
    if (block_table.dtype is not _I32 or kv_len.dtype is not _I32 or cu_rows.dtype is not _I32 or
            len(table_shape) != 2):
        raise ValueError("block_table must be int32 [n_seqs, max_pages], kv_len and the row offsets int32")
    n, width = table_shape
    if (kv_len.shape != (n,) or cu_rows.shape != (n + 1,) or not kv_len.is_contiguous() or
            not cu_rows.is_contiguous()):
        raise ValueError("kv_len must be [n_seqs], the row offsets [n_seqs + 1], contiguous")
    tst = block_table.stride()
    if width > 1 and tst[1] != 1:
        raise ValueError("block_table's rows must be contiguous")
    if (dev < 0 or v_pages.get_device() != dev or block_table.get_device() != dev or kv_len.get_device() != dev or
            cu_rows.get_device() != dev):
        raise ValueError("every tensor must be on one CUDA device")
    kv = PagedKv(fmt, n_pages, page, nkv, hd, k_pages.data_ptr(), v_pages.data_ptr(),
                 st[0] if n_pages > 1 else page * row, ks, vs, scale_stride)
    batch = PagedBatch(n, n_tokens, width, cu_rows.data_ptr(), kv_len.data_ptr(), block_table.data_ptr(),
                       tst[0] if n > 1 else width)
    return kv, batch, dev


def _rows(t, name, dev, *shape):
    """The distance between the rows of an FP16 tensor of the given shape, each row contiguous."""
    if t.dtype is not _F16 or t.shape != shape or t.get_device() != dev:
        raise ValueError(f"{name} must be a float16 tensor {list(shape)} on the pages' device")
    st = t.stride()
    inner = 1
    for d in range(len(shape) - 1, 0, -1):
        if st[d] != inner and shape[d] != 1:
            raise ValueError(f"{name}'s rows must be contiguous")
        inner *= shape[d]
    return st[0] if shape[0] > 1 else inner


def _packed(t, name, dev, *shape):
    """t, checked to be a contiguous FP16 tensor of the given shape."""
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    _rows(t, name, dev, *shape)
    return t


@contextlib.contextmanager
def _elsewhere(dev, stream):
    """A device that is not current, or a stream that is given, made current: what is allocated belongs to it."""
    with torch.cuda.device(dev), torch.cuda.stream(stream):
        yield


def paged_kv_write(qkv, k_pages, v_pages, block_table, kv_len, cu_rows, *, n_heads, cos=None, sin=None, k_scale=None,
                   v_scale=None, q_out=None, stream=None):
    """Stores a batch's new tokens in their pages (quantised, in 8-bit pages); in place.

    qkv fp16 [T, (n_heads + 2 * n_kv_heads) * head_dim], rows any distance apart.  With
    RoPE tables (fp32 [max_seq, head_dim / 2]) q and k are rotated at the tokens'
    positions; returns q [T, n_heads, head_dim]: rotated in q_out, or without tables
    qkv's own q."""
    T = qkv.shape[0]
    kv, batch, dev = _paged(T, k_pages, v_pages, block_table, kv_len, cu_rows, k_scale, v_scale)
    if stream is not None or dev != torch.cuda.current_device():
        with _elsewhere(dev, stream):
            return paged_kv_write(qkv, k_pages, v_pages, block_table, kv_len, cu_rows, n_heads=n_heads, cos=cos,
                                  sin=sin, k_scale=k_scale, v_scale=v_scale, q_out=q_out)
    hd = kv.head_dim
    stride = _rows(qkv, "qkv", dev, T, (n_heads + 2 * kv.n_kv_heads) * hd)
    c = s = q = None
    max_seq = 0
    if cos is None or sin is None:
        if cos is not None or sin is not None:
            raise ValueError("cos and sin come together")
        if q_out is not None:
            raise ValueError("q_out needs cos and sin: without them q is left in qkv")
    else:
        shape = cos.shape
        if (cos.dtype is not _F32 or sin.dtype is not _F32 or len(shape) != 2 or shape[1] * 2 != hd or
                sin.shape != shape or cos.get_device() != dev or sin.get_device() != dev or
                not cos.is_contiguous() or not sin.is_contiguous()):
            raise ValueError("cos and sin must be contiguous float32 [max_seq, head_dim / 2] on the pages' device")
        max_seq, c, s = shape[0], cos.data_ptr(), sin.data_ptr()
        if q_out is None:
            q_out = torch.empty(T, n_heads, hd, dtype=_F16, device=qkv.device)
        else:
            _packed(q_out, "q_out", dev, T, n_heads, hd)
        q = q_out.data_ptr()
    check(lib().af_paged_kv_write(ctypes.byref(kv), ctypes.byref(batch), qkv.data_ptr(), stride, n_heads, c, s,
                                  max_seq, q, torch.cuda.current_stream(dev).cuda_stream), "af_paged_kv_write")
    return qkv[:, :n_heads * hd].unflatten(1, (n_heads, hd)) if q_out is None else q_out


def paged_kv_read(k_pages, v_pages, block_table, kv_len, cu_rows, n_rows, *, k_scale=None, v_scale=None, k_out=None,
                  v_out=None, stream=None):
    """The last cu_rows[b+1] - cu_rows[b] cached positions of each sequence as fp16 (k, v) [n_rows, n_kv_heads, head_dim]."""
    kv, batch, dev = _paged(n_rows, k_pages, v_pages, block_table, kv_len, cu_rows, k_scale, v_scale)
    if stream is not None or dev != torch.cuda.current_device():
        with _elsewhere(dev, stream):
            return paged_kv_read(k_pages, v_pages, block_table, kv_len, cu_rows, n_rows, k_scale=k_scale,
                                 v_scale=v_scale, k_out=k_out, v_out=v_out)
    shape = (n_rows, kv.n_kv_heads, kv.head_dim)
    k = torch.empty(shape, dtype=_F16, device=k_pages.device) if k_out is None else _packed(k_out, "k_out", dev, *shape)
    v = torch.empty(shape, dtype=_F16, device=k_pages.device) if v_out is None else _packed(v_out, "v_out", dev, *shape)
    check(lib().af_paged_kv_read(ctypes.byref(kv), ctypes.byref(batch), k.data_ptr(), v.data_ptr(),
                                 torch.cuda.current_stream(dev).cuda_stream), "af_paged_kv_read")
    return k, v


def paged_attention(q, k_pages, v_pages, block_table, kv_len, cu_rows, *, scale=None, k_scale=None, v_scale=None,
                    max_q=None, max_kv=None, out=None, stream=None):
    """Causal attention of a batch's new tokens over their cached positions, themselves included.

    q fp16 [T, n_heads, head_dim], tokens any distance apart; returns out, alike and
    contiguous.  scale: 1 / sqrt(head_dim) unless given.  max_q, max_kv: the host's bounds on
    any sequence's new tokens and cached positions, which choose the split of the work."""
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("q must be [T, n_heads, head_dim]")
    T, nh, hd = shape
    kv, batch, dev = _paged(T, k_pages, v_pages, block_table, kv_len, cu_rows, k_scale, v_scale)
    if stream is not None or dev != torch.cuda.current_device():
        with _elsewhere(dev, stream):
            return paged_attention(q, k_pages, v_pages, block_table, kv_len, cu_rows, scale=scale, k_scale=k_scale,
                                   v_scale=v_scale, max_q=max_q, max_kv=max_kv, out=out)
    stride = _rows(q, "q", dev, T, nh, kv.head_dim)
    if out is None:
        out = torch.empty(shape, dtype=_F16, device=q.device)
    else:
        _packed(out, "out", dev, T, nh, hd)
    L, k, b = lib(), ctypes.byref(kv), ctypes.byref(batch)
    # scratch of this call alone, from the stream's allocator: calls on several streams, or in several graphs, share none
    need = L.af_paged_attention_workspace_bytes(k, b, nh, max_q or 0, max_kv or 0)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    check(L.af_paged_attention(k, b, q.data_ptr(), stride, nh, hd ** -0.5 if scale is None else scale, max_q or 0,
                               max_kv or 0, out.data_ptr(), ws.data_ptr() if need else None, need,
                               torch.cuda.current_stream(dev).cuda_stream), "af_paged_attention")
    return out
