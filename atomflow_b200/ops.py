"""Host-side operators over the C ABI, for callers that hold torch CUDA tensors.

PyTorch here is plumbing (device memory, the current stream); all arithmetic
runs in libatomflow_b200.so.  Each op mirrors a reference launcher:

  w8a16_gemv  <- launch_w8a16_gemv   (include/ops/kernel.h:138-145)
  lm_head     <- engine.cu:494-513 cublasGemmEx + argmax launch (engine.cu:521)
  argmax      <- launch_argmax       (include/ops/kernel.h:155-159)

The paged_* ops have no reference launcher: a batch of sequences over a KV
cache in pages (FP16, FP8-E4M3 or INT8), described in include/atomflow_b200.h.
"""
import torch

from ._lib import ArgmaxMode, ScaleKind, WeightDtype, check, lib


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
# Checks, outputs and the call of the C ABI are in the module _torch_ops (csrc/af_torch.cpp): a decode step calls these
# for every layer, and in Python they took longer than the kernels.
#
# stream: a torch.cuda.Stream of the pages' device, the current one unless given.  As with the other ops nothing is
# recorded on it: the caller orders it behind the streams that made the inputs and keeps those alive until it is done; new
# outputs are allocated on it.  No gradients: inputs, tables and given outputs that ask for one are refused.
_native = None


def _paged_ops():
    global _native
    if _native is None:
        lib()   # raises if the library is missing, and loads what the module links to
        try:
            from . import _torch_ops
        except ImportError as e:
            raise ImportError("atomflow_b200/_torch_ops.so is missing or does not fit this torch; build it with "
                              f"`python -m atomflow_b200.build` ({e})") from e
        _native = _torch_ops
    return _native


def _on_stream(stream, device):
    if stream.device != device:
        raise ValueError("the stream must be of the pages' device")
    return torch.cuda.stream(stream)


def paged_kv_write(qkv, k_pages, v_pages, block_table, kv_len, cu_rows, *, n_heads, cos=None, sin=None, k_scale=None,
                   v_scale=None, q_out=None, stream=None):
    """Stores a batch's new tokens in their pages (quantised, in 8-bit pages); in place.

    qkv fp16 [T, (n_heads + 2 * n_kv_heads) * head_dim], rows any multiple of 8 elements apart.  With
    RoPE tables (fp32 [max_seq, head_dim / 2]) q and k are rotated at the tokens'
    positions; returns q [T, n_heads, head_dim]: rotated in q_out, or without tables
    qkv's own q.  The cache and the batch (int32 block_table [n_seqs, max_pages], kv_len
    [n_seqs], cu_rows [n_seqs + 1] on the device) are described in
    include/atomflow_b200.h; pages are fp16, float8_e4m3fn or int8 [n_pages, page_size,
    n_kv_heads, head_dim], the last two with fp16 scales [n_pages, page_size, n_kv_heads]."""
    if stream is not None:
        with _on_stream(stream, k_pages.device):
            return paged_kv_write(qkv, k_pages, v_pages, block_table, kv_len, cu_rows, n_heads=n_heads, cos=cos,
                                  sin=sin, k_scale=k_scale, v_scale=v_scale, q_out=q_out)
    q = (_native or _paged_ops()).paged_kv_write(qkv, k_pages, v_pages, block_table, kv_len, cu_rows, n_heads, cos, sin,
                                                 k_scale, v_scale, q_out)
    if type(q) is int:
        check(q, "af_paged_kv_write")
    return qkv[:, :n_heads * k_pages.shape[3]].unflatten(1, (n_heads, k_pages.shape[3])) if q is None else q


def paged_kv_read(k_pages, v_pages, block_table, kv_len, cu_rows, n_rows, *, k_scale=None, v_scale=None, k_out=None,
                  v_out=None, stream=None):
    """The last cu_rows[b+1] - cu_rows[b] cached positions of each sequence as fp16 (k, v) [n_rows, n_kv_heads, head_dim]."""
    if stream is not None:
        with _on_stream(stream, k_pages.device):
            return paged_kv_read(k_pages, v_pages, block_table, kv_len, cu_rows, n_rows, k_scale=k_scale,
                                 v_scale=v_scale, k_out=k_out, v_out=v_out)
    kv = (_native or _paged_ops()).paged_kv_read(k_pages, v_pages, block_table, kv_len, cu_rows, n_rows, k_scale, v_scale,
                                                 k_out, v_out)
    if type(kv) is int:
        check(kv, "af_paged_kv_read")
    return kv


def paged_attention(q, k_pages, v_pages, block_table, kv_len, cu_rows, *, scale=None, k_scale=None, v_scale=None,
                    max_q=None, max_kv=None, out=None, stream=None):
    """Causal attention of a batch's new tokens over their cached positions, themselves included.

    q fp16 [T, n_heads, head_dim], tokens any multiple of 8 elements apart; returns out, alike and
    contiguous.  scale: 1 / sqrt(head_dim) unless given.  max_q, max_kv: the host's bounds on
    any sequence's new tokens and cached positions, which choose the split of the work (a sequence
    of more tokens than max_q may be left out, which af_device_faults tells)."""
    if stream is not None:
        with _on_stream(stream, k_pages.device):
            return paged_attention(q, k_pages, v_pages, block_table, kv_len, cu_rows, scale=scale, k_scale=k_scale,
                                   v_scale=v_scale, max_q=max_q, max_kv=max_kv, out=out)
    o = (_native or _paged_ops()).paged_attention(q, k_pages, v_pages, block_table, kv_len, cu_rows, scale, k_scale,
                                                  v_scale, max_q, max_kv, out)
    if type(o) is int:
        check(o, "af_paged_attention")
    return o
