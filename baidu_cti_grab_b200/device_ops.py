"""torch-facing wrappers of the C ABI: validate tensors, pass device pointers
and the current stream, allocate outputs with torch's caching allocator.

These are the only functions in the package that call into librep_b200.so;
the reference-shaped modules (w8a8_triton_kernels, quantization,
rep_encoder_fusion, rep_encoder) are built on them.
"""

from __future__ import annotations

import ctypes
import operator
import weakref
from array import array
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import _lib as L

_DT = {
    torch.float32: L.RB_F32,
    torch.bfloat16: L.RB_BF16,
    torch.float16: L.RB_F16,
    torch.int32: L.RB_I32,
    torch.int8: L.RB_I8,
}


def rb_dtype(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype}") from None


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# the current stream's handle without the Stream object around it (2 us less per call), where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def require_cuda(name: str, *tensors: Optional[torch.Tensor]) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} expects CUDA tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"{name}: tensors on different devices ({dev} vs {t.device})")
    if dev is None:
        raise RuntimeError(f"{name} expects CUDA tensors")
    return dev


# --------------------------------------------------------------- RepEncoder
_DERIVED: dict = {}


def cached_derived(src: torch.Tensor, tag: str, make):
    """``make(src)`` computed once per (tensor object, tag) and reused while the
    tensor is alive and unmodified (same storage pointer and version counter).
    Entries die with their source tensor, so a new tensor that happens to
    reuse a freed address never sees a stale value."""
    key = (id(src), tag)
    sig = (src.data_ptr(), src._version, src.dtype, tuple(src.shape), tuple(src.stride()), src.device)
    hit = _DERIVED.get(key)
    if hit is not None:
        ref, hsig, value = hit
        if ref() is src and hsig == sig:
            return value
    value = make(src)
    try:
        ref = weakref.ref(src, lambda _r, k=key: _DERIVED.pop(k, None))
    except TypeError:
        return value
    _DERIVED[key] = (ref, sig, value)
    return value


def _affine_param(t: torch.Tensor) -> torch.Tensor:
    """A LayerNorm parameter as the kernels read it: bf16, fp16 or fp32,
    contiguous (other dtypes are widened to fp32 once and cached).  16-bit
    parameters are read as they are: half the bytes of an fp32 copy."""
    if t.dtype in (torch.bfloat16, torch.float16, torch.float32):
        return t.contiguous()
    return cached_derived(t, "affine_f32", lambda x: x.detach().float().contiguous())


def rep_gather_ln_quant(table: torch.Tensor, slot_values: Sequence[torch.Tensor],
                        slot_offsets: Sequence[torch.Tensor], gamma: torch.Tensor, beta: torch.Tensor,
                        eps: float, act_mode: str = "dynamic", static_scale: Optional[torch.Tensor] = None,
                        q_out: Optional[torch.Tensor] = None, scale_out: Optional[torch.Tensor] = None,
                        want_pooled: bool = False, want_ln: bool = False):
    """Fused gather -> pool -> concat -> LayerNorm -> int8 (rb_rep_gather_ln_quant_idx).

    Slot values and offsets are all int64 (the reference's collate output) or all
    int32 (half the bytes; ids, offsets and nnz below 2^31).
    Returns (q int8[N, S*512] or None, scale fp32[N] or None, pooled or None, ln or None)."""
    S = len(slot_values)
    dev = require_cuda("rep_gather_ln_quant", table, gamma, beta, *slot_values, *slot_offsets)
    if len(slot_offsets) != S:
        raise ValueError("slot_values and slot_offsets differ in length")
    if table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous [V, 512] tensor")
    n_items = int(slot_offsets[0].numel()) - 1 if S else 0
    idx_dtype = slot_offsets[0].dtype if S else torch.int64
    if idx_dtype not in (torch.int64, torch.int32):
        raise ValueError("slot values and offsets must be int64 or int32")
    for s in range(S):
        if slot_values[s].dtype != idx_dtype or slot_offsets[s].dtype != idx_dtype:
            raise ValueError("slot values and offsets must all be int64 or all int32")
        if not slot_values[s].is_contiguous() or not slot_offsets[s].is_contiguous():
            raise ValueError("slot values and offsets must be contiguous")
        if slot_offsets[s].numel() - 1 != n_items:
            raise ValueError("every slot needs offsets of length N+1")
    H = S * table.shape[1]
    mode = {"dynamic": L.RB_ACT_DYNAMIC, "static": L.RB_ACT_STATIC, "none": L.RB_ACT_NONE}[act_mode]
    q = scale = None
    if mode != L.RB_ACT_NONE:
        q = torch.empty((n_items, H), dtype=torch.int8, device=dev) if q_out is None else q_out
        if mode == L.RB_ACT_DYNAMIC:
            scale = torch.empty((n_items,), dtype=torch.float32, device=dev) if scale_out is None else scale_out
    pooled = torch.empty((n_items, H), dtype=table.dtype, device=dev) if want_pooled else None
    ln = torch.empty((n_items, H), dtype=table.dtype, device=dev) if (want_ln or mode == L.RB_ACT_NONE) else None
    gamma = _affine_param(gamma)
    beta = _affine_param(beta)
    if static_scale is not None:
        static_scale = static_scale.contiguous()
    with torch.cuda.device(dev):
        L.call("rb_rep_gather_ln_quant_idx", table.data_ptr(), rb_dtype(table), table.shape[0], table.shape[1],
               L.RB_I32 if idx_dtype == torch.int32 else L.RB_I64,
               L.ptr_array([v.data_ptr() for v in slot_values]),
               L.ptr_array([o.data_ptr() for o in slot_offsets]),
               L.i64_array([v.numel() for v in slot_values]), S, n_items,
               gamma.data_ptr(), beta.data_ptr(), rb_dtype(gamma), float(eps), mode,
               _ptr(static_scale), rb_dtype(static_scale) if static_scale is not None else 0,
               _ptr(q), H if q is None else q.stride(0), _ptr(scale), _ptr(pooled), _ptr(ln), _stream(dev))
    return q, scale, pooled, ln


def rep_gather_pool(table: torch.Tensor, slot_values: Sequence[torch.Tensor],
                    slot_offsets: Sequence[torch.Tensor], col_slot: Sequence[int], width_slots: int,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gather + sum-pool of a subset of slots into columns col_slot[j]*512 of [N, width_slots*512]."""
    S = len(slot_values)
    dev = require_cuda("rep_gather_pool", table, *slot_values, *slot_offsets)
    n_items = int(slot_offsets[0].numel()) - 1
    D = table.shape[1]
    if out is None:
        out = torch.empty((n_items, width_slots * D), dtype=table.dtype, device=dev)
    with torch.cuda.device(dev):
        L.call("rb_rep_gather_pool", table.data_ptr(), rb_dtype(table), table.shape[0], D,
               L.ptr_array([v.data_ptr() for v in slot_values]),
               L.ptr_array([o.data_ptr() for o in slot_offsets]),
               L.i64_array([v.numel() for v in slot_values]), L.i32_array(col_slot), S, n_items,
               out.data_ptr(), out.stride(0), _stream(dev))
    return out


def rep_gather_pool_scatter(table: torch.Tensor, slot_values: Sequence[torch.Tensor],
                            slot_offsets: Sequence[torch.Tensor], col_slot: Sequence[int], dest: Sequence[int],
                            dest_begin: Sequence[int], ld: int, item_shift: int = 0) -> None:
    """Gather + sum-pool of a subset of slots, item i written to the rank that owns
    it: dest[d] + (i - dest_begin[d])*ld + col_slot[j]*512 (elements) for
    dest_begin[d] <= i < dest_begin[d+1] (rb_rep_gather_pool_scatter).  ``dest``
    holds raw device addresses, local or mapped from another GPU (ipc_import).
    Items are processed from ``item_shift`` on, wrapping around."""
    S = len(slot_values)
    dev = require_cuda("rep_gather_pool_scatter", table, *slot_values, *slot_offsets)
    n_items = int(slot_offsets[0].numel()) - 1
    if len(dest) + 1 != len(dest_begin):
        raise ValueError("dest_begin needs len(dest) + 1 entries")
    with torch.cuda.device(dev):
        L.call("rb_rep_gather_pool_scatter", table.data_ptr(), rb_dtype(table), table.shape[0], table.shape[1],
               L.ptr_array([v.data_ptr() for v in slot_values]),
               L.ptr_array([o.data_ptr() for o in slot_offsets]),
               L.i64_array([v.numel() for v in slot_values]), L.i32_array(col_slot), S, n_items,
               L.ptr_array(list(dest)), L.i64_array(dest_begin), len(dest), int(ld),
               int(item_shift) if n_items else 0, _stream(dev))


def ipc_export(t: torch.Tensor):
    """(64-byte CUDA IPC handle of the allocation holding t, t's byte offset in it)."""
    require_cuda("ipc_export", t)
    handle = (ctypes.c_char * L.RB_IPC_HANDLE_BYTES)()
    off = ctypes.c_int64(0)
    with torch.cuda.device(t.device):
        L.call("rb_ipc_export", t.data_ptr(), handle, ctypes.byref(off))
    return bytes(handle), int(off.value)


def ipc_import(handle: bytes, offset: int, device: torch.device) -> int:
    """Device address, in this process, of another process's exported buffer."""
    if len(handle) != L.RB_IPC_HANDLE_BYTES:
        raise ValueError("an IPC handle has 64 bytes")
    ptr = ctypes.c_void_p(0)
    buf = (ctypes.c_char * L.RB_IPC_HANDLE_BYTES).from_buffer_copy(handle)
    with torch.cuda.device(device):
        L.call("rb_ipc_import", buf, int(offset), ctypes.byref(ptr))
    return int(ptr.value)


def ipc_close(ptr: int, offset: int, device: torch.device) -> None:
    with torch.cuda.device(device):
        L.call("rb_ipc_close", ptr, int(offset))


def layernorm_quant(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float,
                    act_mode: str = "dynamic", static_scale: Optional[torch.Tensor] = None,
                    want_ln: bool = False):
    """LayerNorm (+ int8 quantisation) of dense rows x[N, S*512] (rb_layernorm_quant)."""
    dev = require_cuda("layernorm_quant", x, gamma, beta)
    if x.dim() != 2 or x.shape[1] % 512 != 0:
        raise ValueError("layernorm_quant expects x as [N, S*512]")
    if x.stride(1) != 1:
        x = x.contiguous()
    n, H = x.shape
    S = H // 512
    mode = {"dynamic": L.RB_ACT_DYNAMIC, "static": L.RB_ACT_STATIC, "none": L.RB_ACT_NONE}[act_mode]
    q = torch.empty((n, H), dtype=torch.int8, device=dev) if mode != L.RB_ACT_NONE else None
    scale = torch.empty((n,), dtype=torch.float32, device=dev) if mode == L.RB_ACT_DYNAMIC else None
    ln = torch.empty((n, H), dtype=x.dtype, device=dev) if (want_ln or mode == L.RB_ACT_NONE) else None
    gamma = _affine_param(gamma)
    beta = _affine_param(beta)
    if static_scale is not None:
        static_scale = static_scale.contiguous()
    with torch.cuda.device(dev):
        L.call("rb_layernorm_quant", x.data_ptr(), rb_dtype(x), n, S, x.stride(0), gamma.data_ptr(),
               beta.data_ptr(), rb_dtype(gamma), float(eps), mode, _ptr(static_scale),
               rb_dtype(static_scale) if static_scale is not None else 0, _ptr(q), H, _ptr(scale), _ptr(ln),
               _stream(dev))
    return q, scale, ln


def layernorm_quant_slots(slot_rows: Sequence[torch.Tensor], gamma: torch.Tensor, beta: torch.Tensor, eps: float,
                          act_mode: str = "dynamic", static_scale: Optional[torch.Tensor] = None,
                          want_ln: bool = False):
    """LayerNorm (+ int8) of rows whose slot s is the [N, 512] view slot_rows[s] (common row stride)."""
    dev = require_cuda("layernorm_quant_slots", gamma, beta, *slot_rows)
    S = len(slot_rows)
    n = slot_rows[0].shape[0]
    ld = slot_rows[0].stride(0)
    for v in slot_rows:
        if tuple(v.shape) != (n, 512) or v.stride() != (ld, 1) or v.dtype != slot_rows[0].dtype:
            raise ValueError("slot rows must be [N, 512] views with one common row stride and dtype")
    H = S * 512
    mode = {"dynamic": L.RB_ACT_DYNAMIC, "static": L.RB_ACT_STATIC, "none": L.RB_ACT_NONE}[act_mode]
    q = torch.empty((n, H), dtype=torch.int8, device=dev) if mode != L.RB_ACT_NONE else None
    scale = torch.empty((n,), dtype=torch.float32, device=dev) if mode == L.RB_ACT_DYNAMIC else None
    ln = torch.empty((n, H), dtype=slot_rows[0].dtype, device=dev) if (want_ln or mode == L.RB_ACT_NONE) else None
    gamma = _affine_param(gamma)
    beta = _affine_param(beta)
    if static_scale is not None:
        static_scale = static_scale.contiguous()
    with torch.cuda.device(dev):
        L.call("rb_layernorm_quant_slots", L.ptr_array([v.data_ptr() for v in slot_rows]), rb_dtype(slot_rows[0]),
               n, S, ld, gamma.data_ptr(), beta.data_ptr(), rb_dtype(gamma), float(eps), mode, _ptr(static_scale),
               rb_dtype(static_scale) if static_scale is not None else 0, _ptr(q), H, _ptr(scale), _ptr(ln),
               _stream(dev))
    return q, scale, ln


# ------------------------------------------------------------- quantisers
def quant_dynamic_per_token_out(x2d: torch.Tensor, xq: torch.Tensor, scale: torch.Tensor):
    dev = require_cuda("dynamic_per_token_quantize_activation", x2d, xq, scale)
    if x2d.dim() != 2 or x2d.stride(1) != 1 or xq.stride(1) != 1:
        raise ValueError("expected 2-D row-major x and xq")
    M, K = x2d.shape
    with torch.cuda.device(dev):
        L.call("rb_quant_dynamic_per_token", x2d.data_ptr(), rb_dtype(x2d), M, K, x2d.stride(0), xq.data_ptr(),
               xq.stride(0), scale.data_ptr(), _stream(dev))
    return xq, scale


def quant_static_out(x: torch.Tensor, scale: torch.Tensor, xq: torch.Tensor) -> torch.Tensor:
    dev = require_cuda("static_quantize_activation", x, scale, xq)
    if not x.is_contiguous() or not xq.is_contiguous():
        raise ValueError("static quantisation expects contiguous tensors")
    with torch.cuda.device(dev):
        L.call("rb_quant_static", x.data_ptr(), rb_dtype(x), x.numel(), scale.data_ptr(), rb_dtype(scale),
               xq.data_ptr(), _stream(dev))
    return xq


def quant_rows_v1(x2d: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    dev = require_cuda("quantize_rows_int8", x2d)
    M, K = x2d.shape
    q = torch.empty((M, K), dtype=torch.int8, device=dev)
    s = torch.empty((M,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        L.call("rb_quant_rows_v1", x2d.data_ptr(), rb_dtype(x2d), M, K, x2d.stride(0), q.data_ptr(), K,
               s.data_ptr(), _stream(dev))
    return q, s


def quantize_weight_per_channel(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """W[N,K] -> (q int8 [N,K] K-contiguous, scale fp32 [N])."""
    dev = require_cuda("quantize_weight_per_channel", w)
    if w.dim() != 2:
        raise ValueError("expected W as [N, K]")
    if w.stride(1) != 1:
        w = w.contiguous()
    N, K = w.shape
    q = torch.empty((N, K), dtype=torch.int8, device=dev)
    s = torch.empty((N,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        L.call("rb_quantize_weight_per_channel", w.data_ptr(), rb_dtype(w), N, K, w.stride(0), q.data_ptr(),
               s.data_ptr(), _stream(dev))
    return q, s


def pack_weight_nk(qweight_t: torch.Tensor) -> torch.Tensor:
    """[K,N] int8 view (any strides) -> [N,K] K-contiguous int8 copy."""
    dev = require_cuda("pack_weight_nk", qweight_t)
    K, N = qweight_t.shape
    dst = torch.empty((N, K), dtype=torch.int8, device=dev)
    with torch.cuda.device(dev):
        L.call("rb_pack_weight_nk", qweight_t.data_ptr(), K, N, qweight_t.stride(0), qweight_t.stride(1),
               dst.data_ptr(), _stream(dev))
    return dst


def as_nk(qweight_t: torch.Tensor) -> torch.Tensor:
    """The K-contiguous [N,K] view of a [K,N] weight, repacking only when needed."""
    K, N = qweight_t.shape
    if qweight_t.stride(0) == 1 and qweight_t.stride(1) >= K and qweight_t.stride(1) % 16 == 0 \
            and qweight_t.data_ptr() % 16 == 0:
        return qweight_t.t()
    return pack_weight_nk(qweight_t)


# ------------------------------------------------------------------- GEMM
_WS_SIZE: Dict[Tuple[int, int, int], int] = {}
_WS: Dict[Tuple[int, int], torch.Tensor] = {}


def _workspace_elems(M: int, N: int, K: int) -> int:
    key = (M, N, K)
    n = _WS_SIZE.get(key)
    if n is None:
        n = _WS_SIZE[key] = int(L.load().rb_w8a8_gemm_workspace_size(M, N, K))
    return n


def _workspace(dev: torch.device, elems: int) -> torch.Tensor:
    """The split-K workspace of the current stream on `dev`, grown on demand.
    One buffer per (device, stream): launches on one stream run in order, so
    consecutive GEMMs on a stream can share it."""
    key = (dev.index, torch.cuda.current_stream(dev).cuda_stream)
    ws = _WS.get(key)
    if ws is None or ws.numel() < elems:
        ws = _WS[key] = torch.empty((elems,), dtype=torch.int32, device=dev)
    return ws


def w8a8_gemm(a: torch.Tensor, b_nk: torch.Tensor, scale_a: Optional[torch.Tensor],
              scale_b: Optional[torch.Tensor], out: torch.Tensor, *, bias: Optional[torch.Tensor] = None,
              sa_per_row: bool = True) -> torch.Tensor:
    """out = ((f32(A @ B^T) * sa) * sb) + bias, or raw int32 when out is int32."""
    dev = require_cuda("w8a8_gemm", a, b_nk, out, scale_a, scale_b, bias)
    if a.dim() != 2 or b_nk.dim() != 2 or a.stride(1) != 1 or b_nk.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("w8a8_gemm expects row-major 2-D operands")
    M, K = a.shape
    N = b_nk.shape[0]
    if b_nk.shape[1] != K:
        raise ValueError(f"shape mismatch: A K={K}, B K={b_nk.shape[1]}")
    if tuple(out.shape) != (M, N):
        raise ValueError(f"out must be [{M}, {N}]")
    raw = out.dtype == torch.int32
    if not raw:
        scale_a = scale_a.contiguous()
        scale_b = scale_b.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    ws_elems = _workspace_elems(M, N, K)
    ws = _workspace(dev, ws_elems) if ws_elems > 0 else None
    with torch.cuda.device(dev):
        L.call("rb_w8a8_gemm_ws", a.data_ptr(), a.stride(0), b_nk.data_ptr(), b_nk.stride(0), M, N, K,
               _ptr(scale_a), rb_dtype(scale_a) if scale_a is not None else 0, 1 if sa_per_row else 0,
               _ptr(scale_b), rb_dtype(scale_b) if scale_b is not None else 0, _ptr(bias),
               rb_dtype(bias) if bias is not None else 0, out.data_ptr(), out.stride(0), rb_dtype(out),
               _ptr(ws), ws_elems, _stream(dev))
    return out


def w8a8_gemm_ln(a: torch.Tensor, b_nk: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
                 out: torch.Tensor, ln_gamma: torch.Tensor, ln_beta: torch.Tensor, eps: float, ln_out: torch.Tensor,
                 *, bias: Optional[torch.Tensor] = None, sa_per_row: bool = True):
    """out = ((f32(A @ B^T) * sa) * sb) + bias and ln_out = LayerNorm(out) over its 512
    columns (rb_w8a8_gemm_ln).  Returns (out, ln_out)."""
    dev = require_cuda("w8a8_gemm_ln", a, b_nk, out, ln_out, scale_a, scale_b, bias, ln_gamma, ln_beta)
    if a.dim() != 2 or b_nk.dim() != 2 or a.stride(1) != 1 or b_nk.stride(1) != 1 or out.stride(1) != 1 \
            or ln_out.stride(1) != 1:
        raise ValueError("w8a8_gemm_ln expects row-major 2-D operands")
    M, K = a.shape
    N = b_nk.shape[0]
    if b_nk.shape[1] != K:
        raise ValueError(f"shape mismatch: A K={K}, B K={b_nk.shape[1]}")
    if tuple(out.shape) != (M, N) or tuple(ln_out.shape) != (M, N) or ln_out.dtype != out.dtype:
        raise ValueError(f"out and ln_out must be [{M}, {N}] of one dtype")
    scale_a, scale_b = scale_a.contiguous(), scale_b.contiguous()
    bias = None if bias is None else bias.contiguous()
    ln_gamma, ln_beta = ln_gamma.contiguous(), ln_beta.contiguous()
    with torch.cuda.device(dev):
        L.call("rb_w8a8_gemm_ln", a.data_ptr(), a.stride(0), b_nk.data_ptr(), b_nk.stride(0), M, N, K,
               scale_a.data_ptr(), rb_dtype(scale_a), 1 if sa_per_row else 0, scale_b.data_ptr(), rb_dtype(scale_b),
               _ptr(bias), rb_dtype(bias) if bias is not None else 0, out.data_ptr(), out.stride(0), rb_dtype(out),
               ln_gamma.data_ptr(), ln_beta.data_ptr(), rb_dtype(ln_gamma), float(eps), ln_out.data_ptr(),
               ln_out.stride(0), _stream(dev))
    return out, ln_out


def fp_gemm(a: torch.Tensor, b_nk: torch.Tensor, out: torch.Tensor, *,
            bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = A @ B^T + bias on the tensor cores: A [M, K], B [N, K] both bf16
    (kind::f16) or both fp32 (kind::tf32), fp32 accumulation."""
    dev = require_cuda("fp_gemm", a, b_nk, out, bias)
    if a.dim() != 2 or b_nk.dim() != 2 or a.stride(1) != 1 or b_nk.stride(1) != 1 or out.stride(1) != 1:
        raise ValueError("fp_gemm expects row-major 2-D operands")
    if a.dtype != b_nk.dtype or a.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("fp_gemm operands must both be bf16 or both fp32")
    M, K = a.shape
    N = b_nk.shape[0]
    if b_nk.shape[1] != K:
        raise ValueError(f"shape mismatch: A K={K}, B K={b_nk.shape[1]}")
    if tuple(out.shape) != (M, N):
        raise ValueError(f"out must be [{M}, {N}]")
    if bias is not None:
        bias = bias.contiguous()
    with torch.cuda.device(dev):
        L.call("rb_fp_gemm", a.data_ptr(), rb_dtype(a), a.stride(0), b_nk.data_ptr(), b_nk.stride(0), M, N, K,
               _ptr(bias), rb_dtype(bias) if bias is not None else 0, out.data_ptr(), out.stride(0), rb_dtype(out),
               _stream(dev))
    return out


_SMOE_WS: Dict[Tuple[int, int], torch.Tensor] = {}


def smoe_experts(x: torch.Tensor, topk_idx: torch.Tensor, topk_score: torch.Tensor, w1: torch.Tensor,
                 b1: Optional[torch.Tensor], w2: torch.Tensor, b2: Optional[torch.Tensor],
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The SMoE expert layer after the gate (rb_smoe_experts).

    x [T, D] bf16/f16; topk_idx [T, k] int64/int32; topk_score [T, k] in x.dtype;
    w1 [E, F, D], b1 [E, F], w2 [E, D, F], b2 [E, D] in x.dtype.
    Returns out [T, D] = sum over each token's k experts of
    score * (relu(x W1^T + b1) W2^T + b2)."""
    dev = require_cuda("smoe_experts", x, topk_idx, topk_score, w1, b1, w2, b2, out)
    if x.dim() != 2 or topk_idx.dim() != 2 or topk_score.shape != topk_idx.shape:
        raise ValueError("smoe_experts expects x [T, D] and topk_idx/topk_score [T, k]")
    T, D = x.shape
    k = topk_idx.shape[1]
    if topk_idx.shape[0] != T:
        raise ValueError("topk_idx must have one row per token")
    if w1.dim() != 3 or w2.dim() != 3 or w1.shape[2] != D or w2.shape[1] != D or w2.shape[0] != w1.shape[0] \
            or w2.shape[2] != w1.shape[1]:
        raise ValueError("w1 must be [E, F, D] and w2 [E, D, F]")
    E, F = w1.shape[0], w1.shape[1]
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("smoe_experts takes bf16 or f16 activations")
    if topk_idx.dtype not in (torch.int64, torch.int32):
        raise ValueError("topk_idx must be int64 or int32")
    if any(t is not None and t.dtype != x.dtype for t in (topk_score, w1, b1, w2, b2)):
        raise ValueError("scores, weights and biases must share x's dtype")
    if x.stride(1) != 1:
        x = x.contiguous()
    topk_idx, topk_score = topk_idx.contiguous(), topk_score.contiguous()
    w1, w2 = w1.contiguous(), w2.contiguous()
    b1 = None if b1 is None else b1.contiguous()
    b2 = None if b2 is None else b2.contiguous()
    if out is None:
        out = torch.empty((T, D), dtype=x.dtype, device=dev)
    elif tuple(out.shape) != (T, D) or out.dtype != x.dtype or out.stride(1) != 1:
        raise ValueError(f"out must be a row-major [{T}, {D}] {x.dtype} tensor")
    lib = L.load()
    idt = L.RB_I64 if topk_idx.dtype == torch.int64 else L.RB_I32
    need = int(lib.rb_smoe_workspace_size(T, k, E, D, F, rb_dtype(x)))
    if need < 0:
        raise ValueError("rb_smoe_workspace_size rejected the shape")
    key = (dev.index, torch.cuda.current_stream(dev).cuda_stream)
    ws = _SMOE_WS.get(key)
    if ws is None or ws.numel() < need:
        ws = _SMOE_WS[key] = torch.empty((max(need, 256),), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        L.call("rb_smoe_experts", x.data_ptr(), rb_dtype(x), x.stride(0), T, D, topk_idx.data_ptr(), idt,
               topk_score.data_ptr(), k, E, w1.data_ptr(), _ptr(b1), w2.data_ptr(), _ptr(b2), F, ws.data_ptr(),
               ws.numel(), out.data_ptr(), out.stride(0), _stream(dev))
    return out


# ------------------------------------------------------- routing to experts
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_INDEX = {torch.int32: L.RB_I32, torch.int64: L.RB_I64}
_SCORES = {"softmax": L.RB_SCORE_SOFTMAX, "sigmoid": L.RB_SCORE_SIGMOID}


def _call_on(dev: torch.device, name: str, *args) -> None:
    """L.call on `dev`'s current stream, which becomes the last argument."""
    index = dev.index
    if torch.cuda.current_device() == index:
        L.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            L.call(name, *args, _raw_stream(index))


_PLAN_BYTES: Dict[tuple, int] = {}  # workspace bytes of the shapes seen last


def _plan_bytes(dev: torch.device, name: str, *shape: int) -> int:
    """What a workspace-size entry point says of a shape on `dev` (it goes by the device's SMs)."""
    key = (dev.index, name, *shape)
    n = _PLAN_BYTES.get(key)
    if n is None:
        with torch.cuda.device(dev):
            n = int(getattr(L.load(), name)(*shape))
        if n < 0:
            raise ValueError(f"{name} rejected the shape {shape}")
        if len(_PLAN_BYTES) >= 4096:
            _PLAN_BYTES.clear()
        _PLAN_BYTES[key] = n
    return n


def _device_of(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    """require_cuda for a call whose first tensor is always there (a microsecond less)."""
    dev = first.device
    if dev.type != "cuda":
        raise RuntimeError(f"{name} expects CUDA tensors")
    for t in others:
        if t is not None and t.device != dev:
            require_cuda(name, first, t)
    return dev


def _rows_of(t: torch.Tensor, rows: int, width: int) -> Tuple[torch.Tensor, int]:
    """A matrix with contiguous rows (a copy only where t has none) and its row pitch in elements."""
    s0, s1 = t.stride()
    if (s1 != 1 and width > 1) or (rows > 1 and s0 < width):
        t = t.contiguous()
        s0 = width
    return t, max(s0, width)


def route_topk(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
               groups: int = 1, topk_groups: int = 1, group_top: int = 2, renormalize: bool = False,
               scale: float = 1.0, idx_dtype: torch.dtype = torch.int64, score_dtype: Optional[torch.dtype] = None,
               want_probs: bool = False, want_counts: bool = False):
    """The choice of k experts per token that smoe_experts takes (rb_route_topk).

    logits [T, E] fp32/bf16/f16 (rows may be strided), E <= 512, k <= 32; a logit of -inf or of
    the type's lowest value masks its expert.  bias fp32 [E] counts for the choice only.  Of `groups`
    equal runs of experts the topk_groups with the highest sums of their group_top best stay.
    Returns (idx [T, k] by falling choice value, ties to the lowest index; score [T, k] in score_dtype
    (default: the logits'), probs [T, E] in score_dtype or None, counts int32 [E] or None)."""
    dev = _device_of("route_topk", logits, bias)
    dtype = logits.dtype
    if logits.dim() != 2 or dtype not in _FLOATS:
        raise ValueError("route_topk expects logits [T, E] in fp32, bf16 or f16")
    T, E = logits.shape
    kind = _SCORES.get(score)
    if kind is None:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, not {score!r}")
    bias_ptr = None
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (E,):
            raise ValueError(f"bias must be fp32 [{E}]")
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    if idx_dtype is not torch.int64 and idx_dtype is not torch.int32:
        raise ValueError("idx_dtype must be int64 or int32")
    if score_dtype is None:
        score_dtype = dtype
    elif score_dtype not in _FLOATS:
        raise ValueError("score_dtype must be fp32, bf16 or f16")
    if not 1 <= k <= max(E, 1):
        raise ValueError(f"k must be in [1, {E}]")
    logits, ld = _rows_of(logits, T, E)
    idx = torch.empty((T, k), dtype=idx_dtype, device=dev)
    chosen = torch.empty((T, k), dtype=score_dtype, device=dev)
    probs = counts = probs_ptr = counts_ptr = None
    if want_probs:
        probs = torch.empty((T, E), dtype=score_dtype, device=dev)
        probs_ptr = probs.data_ptr()
    if want_counts:
        counts = torch.empty((E,), dtype=torch.int32, device=dev)
        counts_ptr = counts.data_ptr()
    _call_on(dev, "rb_route_topk", logits.data_ptr(), _DT[dtype], ld, T, E, bias_ptr, k, kind, groups, topk_groups,
             group_top, bool(renormalize), float(scale), idx.data_ptr(), L.RB_I64 if idx_dtype is torch.int64 else L.RB_I32,
             chosen.data_ptr(), _DT[score_dtype], probs_ptr, counts_ptr)
    return idx, chosen, probs, counts


def route_topk_backward(logits: torch.Tensor, idx: torch.Tensor, grad_score: Optional[torch.Tensor],
                        grad_probs: Optional[torch.Tensor] = None, *, score: str = "softmax",
                        renormalize: bool = False, scale: float = 1.0) -> torch.Tensor:
    """Gradient [T, E] of route_topk's logits, in their dtype (rb_route_topk_backward), from the
    gradients of its scores [T, k] and probs [T, E] (either may be None) and its idx."""
    dev = _device_of("route_topk_backward", logits, idx, grad_score, grad_probs)
    dtype = logits.dtype
    if logits.dim() != 2 or dtype not in _FLOATS:
        raise ValueError("route_topk_backward expects logits [T, E] in fp32, bf16 or f16")
    T, E = logits.shape
    kind = _SCORES.get(score)
    if kind is None:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, not {score!r}")
    if idx.dim() != 2 or idx.shape[0] != T or idx.dtype not in (torch.int64, torch.int32):
        raise ValueError("idx must be int64 or int32 [T, k]")
    gs_ptr = gp_ptr = None
    gs_type = gp_type = 0
    if grad_score is not None:
        if grad_score.shape != idx.shape or grad_score.dtype not in _FLOATS:
            raise ValueError("grad_score must be a float tensor of idx's shape")
        grad_score = grad_score.contiguous()
        gs_ptr, gs_type = grad_score.data_ptr(), _DT[grad_score.dtype]
    if grad_probs is not None:
        if grad_probs.shape != logits.shape or grad_probs.dtype not in _FLOATS:
            raise ValueError("grad_probs must be a float tensor of the logits' shape")
        grad_probs = grad_probs.contiguous()
        gp_ptr, gp_type = grad_probs.data_ptr(), _DT[grad_probs.dtype]
    logits, ld = _rows_of(logits, T, E)
    idx = idx.contiguous()
    out = torch.empty((T, E), dtype=dtype, device=dev)
    _call_on(dev, "rb_route_topk_backward", logits.data_ptr(), _DT[dtype], ld, T, E, idx.data_ptr(),
             L.RB_I64 if idx.dtype is torch.int64 else L.RB_I32, idx.shape[1], gs_ptr, gs_type, gp_ptr, gp_type, kind,
             bool(renormalize), float(scale), out.data_ptr(), _DT[dtype])
    return out


# -------------------------------------- norms, gate and residual between blocks
_NORMS = {None: L.RB_NORM_NONE, "layer": L.RB_NORM_LAYER, "rms": L.RB_NORM_RMS}
_GATE_ACTS = {"none": L.RB_GATE_ACT_NONE, "sigmoid": L.RB_GATE_ACT_SIGMOID}


def _affine(weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], kind: Optional[str], D: int):
    """(weight pointer, bias pointer, type) of a norm's parameters."""
    dtype = None
    for t in (weight, bias):
        if t is None:
            continue
        if kind is None:
            raise ValueError("a weight or bias was given without its norm")
        if t.shape != (D,) or t.dtype not in _FLOATS or not t.is_contiguous():
            raise ValueError(f"norm weights and biases must be contiguous fp32, bf16 or f16 [{D}]")
        if dtype is not None and t.dtype != dtype:
            raise ValueError("a norm's weight and bias must share a type")
        dtype = t.dtype
    return _ptr(weight), _ptr(bias), 0 if dtype is None else _DT[dtype]


def _norm_args(name, x, h, post, post_weight, post_bias, gate, gate_act, pre, pre_weight, pre_bias):
    """What both directions check: (device, rows, width, x rows, their pitch, h rows, their pitch, gate (kind, tensor, type,
    pitch), post (kind, weight, bias, type), pre likewise, act code)."""
    dev = _device_of(name, x, h, post_weight, post_bias, gate, pre_weight, pre_bias)
    dtype, shape = x.dtype, x.shape
    if dtype not in _FLOATS or len(shape) < 1 or shape != h.shape or h.dtype != dtype:
        raise ValueError(f"{name} expects x and h [..., D] of one shape and one type (fp32, bf16 or f16)")
    k1, k2, act = _NORMS.get(post), _NORMS.get(pre), _GATE_ACTS.get(gate_act)
    if k1 is None or k2 is None:
        raise ValueError("post and pre are 'layer', 'rms' or None")
    if act is None:
        raise ValueError(f"gate_act must be one of {sorted(_GATE_ACTS)}")
    D = shape[-1]
    first, second = (k1, *_affine(post_weight, post_bias, post, D)), (k2, *_affine(pre_weight, pre_bias, pre, D))
    x2, ldx = _rows2d(x, D)
    h2, ldh = _rows2d(h, D)
    g = (L.RB_GATE_NONE, None, 0, 0)
    if gate is not None:
        if gate.dtype not in _FLOATS:
            raise ValueError("the gate must be fp32, bf16 or f16")
        if gate.shape == (D,) and (len(shape) > 1 or D != 1):
            g = (L.RB_GATE_CHANNEL, gate.contiguous(), _DT[gate.dtype], 0)
        elif gate.shape == (*shape[:-1], 1):
            g = (L.RB_GATE_ROW, gate.reshape(-1).contiguous(), _DT[gate.dtype], 1)
        elif gate.shape == shape:
            if gate.dtype != dtype:
                raise ValueError("a gate of every element must have x's type")
            g2, ldg = _rows2d(gate, D)
            g = (L.RB_GATE_FULL, g2, _DT[dtype], ldg)
        else:
            raise ValueError(f"the gate must be [{D}], [..., 1] or of x's shape")
    return dev, x2.shape[0], D, x2, ldx, h2, ldh, g, first, second, act


def _rows2d(t: torch.Tensor, D: int) -> Tuple[torch.Tensor, int]:
    """t [..., D] as rows [N, D] with contiguous values (a copy only where no view has them), and their pitch."""
    if t.dim() != 2:
        t = t.reshape(-1, D) if D else t.reshape(0, 0)
    return _rows_of(t, t.shape[0], D)


def sandwich_norm(x: torch.Tensor, h: torch.Tensor, *, post: Optional[str] = None,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                  post_eps: float = 1e-5, gate: Optional[torch.Tensor] = None, gate_act: str = "none", scale: float = 1.0,
                  pre: Optional[str] = None, pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, pre_eps: float = 1e-5, want_stats: bool = False):
    """The seam between two blocks as one kernel (rb_sandwich_norm): y = x + scale * act(gate) * post(h), z = pre(y).

    x (the residual stream) and h (a block's output) [..., D], D <= 8192; post and pre 'layer', 'rms' or
    None with optional weights and biases [D]; gate None, [D], [..., 1] or x's shape, as it is or its
    sigmoid.  Returns (y, z or None, stats fp32 [N, 4] or None: what sandwich_norm_backward takes)."""
    dev, N, D, x2, ldx, h2, ldh, g, first, second, act = _norm_args("sandwich_norm", x, h, post, post_weight, post_bias,
                                                                    gate, gate_act, pre, pre_weight, pre_bias)
    gk, g2, gt, ldg = g
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    z = torch.empty_like(y) if second[0] != L.RB_NORM_NONE else None
    stats = torch.empty((N, 4), dtype=torch.float32, device=dev) if want_stats else None
    _call_on(dev, "rb_sandwich_norm", x2.data_ptr(), ldx, h2.data_ptr(), ldh, _DT[x.dtype], N, D, *first, float(post_eps), gk,
             _ptr(g2), gt, ldg, act, float(scale), *second, float(pre_eps), y.data_ptr(), _ptr(z), _ptr(stats))
    return y, z, stats


def sandwich_norm_backward(grad_y: Optional[torch.Tensor], grad_z: Optional[torch.Tensor], x: torch.Tensor,
                           h: torch.Tensor, stats: torch.Tensor, *, post: Optional[str] = None,
                           post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                           gate: Optional[torch.Tensor] = None, gate_act: str = "none", scale: float = 1.0,
                           pre: Optional[str] = None, pre_weight: Optional[torch.Tensor] = None,
                           pre_bias: Optional[torch.Tensor] = None):
    """Gradients (x, h, gate, post_weight, post_bias, pre_weight, pre_bias) of sandwich_norm, None where
    there is no such input (rb_sandwich_norm_backward), from those of y and z (either may be None) and the
    forward call's inputs and stats.  The same bits every time."""
    dev, N, D, x2, ldx, h2, ldh, g, first, second, act = _norm_args("sandwich_norm_backward", x, h, post, post_weight,
                                                                    post_bias, gate, gate_act, pre, pre_weight, pre_bias)
    _device_of("sandwich_norm_backward", x, grad_y, grad_z, stats)
    gk, g2, gt, ldg = g
    grads = []
    for t in (grad_y, grad_z):
        if t is None:
            grads += (None, D)
            continue
        if t.shape != x.shape or t.dtype != x.dtype:
            raise ValueError("grad_y and grad_z must have x's shape and type")
        t, ld = _rows2d(t, D)
        grads += (t, ld)
    dy, ldy, dz, ldz = grads
    if dz is not None and pre is None:
        raise ValueError("grad_z was given without pre")
    if stats.shape != (N, 4) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"stats must be the forward call's fp32 [{N}, 4]")
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dh = torch.empty_like(dx)
    outs = [None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)
            for t in (gate, post_weight, post_bias, pre_weight, pre_bias)]
    ws_bytes = _plan_bytes(dev, "rb_sandwich_norm_workspace_size", N, D, _DT[x.dtype])
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    _call_on(dev, "rb_sandwich_norm_backward", _ptr(dy), ldy, _ptr(dz), ldz, x2.data_ptr(), ldx, h2.data_ptr(), ldh,
             stats.data_ptr(), _DT[x.dtype], N, D, *first, gk, _ptr(g2), gt, ldg, act, float(scale), *second, ws.data_ptr(),
             ws_bytes, dx.data_ptr(), dh.data_ptr(), *(_ptr(t) for t in outs))
    return (dx, dh, *outs)


# -------------------------------------------------------- low-rank adapters
def _rows_overlap(a: torch.Tensor, lda: int, b: torch.Tensor, ldb: int) -> bool:
    """Whether two matrices of the same type and height, rows contiguous and lda / ldb apart, share elements (those of
    different pitch in one range of memory are taken to)."""
    (T, wa), wb, size = a.shape, b.shape[1], a.element_size()
    if T == 0 or wa == 0 or wb == 0:
        return False
    d, odd = divmod(b.data_ptr() - a.data_ptr(), size)
    if d >= (T - 1) * lda + wa or -d >= (T - 1) * ldb + wb:
        return False
    return lda != ldb or odd != 0 or not wa <= d % lda <= lda - wb


def low_rank_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter: torch.Tensor,
                 scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] + scale[i] * b[i] @ (a[i] @ x[t]) with i = adapter[t] (rb_low_rank_add): the adapters of many
    requests beside the projection that gave y.

    y [T, N] and x [T, K] bf16/f16; a [R, rank, K] and b [R, N, rank] contiguous in the same type, rank <= 128;
    adapter int32/int64 [T], -1 (or anything outside [0, R)) for a token without one; scale fp32 [R].
    ``out`` may be y, and shares no other memory with y or x.  Forward only: an input that asks for a gradient is refused."""
    dev = _device_of("low_rank_add", y, x, a, b, adapter, scale, out)
    if y.dim() != 2 or x.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError("low_rank_add expects y [T, N], x [T, K], a [R, rank, K] and b [R, N, rank]")
    (T, N), (R, rank, K) = y.shape, a.shape
    if x.shape != (T, K) or b.shape != (R, N, rank):
        raise ValueError(f"x must be [{T}, {K}] and b [{R}, {N}, {rank}]")
    dtype = x.dtype
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or y.dtype is not dtype or a.dtype is not dtype \
            or b.dtype is not dtype:
        raise ValueError("y, x, a and b must all be bf16 or all f16")
    if adapter.shape != (T,) or adapter.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"adapter must be int32 or int64 [{T}]")
    if scale is not None:
        if scale.shape != (R,) or scale.dtype is not torch.float32:
            raise ValueError(f"scale must be fp32 [{R}]")
        scale = scale.contiguous()
    if not a.is_contiguous() or not b.is_contiguous():
        raise ValueError("a and b must be contiguous")
    if torch.is_grad_enabled() and (y.requires_grad or x.requires_grad or a.requires_grad or b.requires_grad
                                    or (scale is not None and scale.requires_grad)
                                    or (out is not None and out.requires_grad)):
        raise RuntimeError("low_rank_add has no backward: call it under torch.no_grad() or on detached tensors")
    given = out is not None
    if not given:
        out = torch.empty((T, N), dtype=dtype, device=dev)
    elif out.shape != (T, N) or out.dtype is not dtype or (N > 1 and out.stride(1) != 1) or (T > 1 and out.stride(0) < N):
        raise ValueError(f"out must be a row-major [{T}, {N}] {dtype} tensor")
    y, ldy = _rows_of(y, T, N)
    x, ldx = _rows_of(x, T, K)
    ldo = max(out.stride(0), N)
    if given:
        in_place = out.data_ptr() == y.data_ptr() and ldo == ldy
        if (not in_place and _rows_overlap(out, ldo, y, ldy)) or _rows_overlap(out, ldo, x, ldx):
            raise ValueError("out may be y itself, and must not overlap y or x elsewhere")
    adapter = adapter.contiguous()
    ws_bytes = _plan_bytes(dev, "rb_low_rank_workspace_size", T, K, N, rank)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev) if ws_bytes else None
    _call_on(dev, "rb_low_rank_add", y.data_ptr(), ldy, x.data_ptr(), ldx, _DT[dtype], T, K, N, a.data_ptr(), b.data_ptr(), R,
             rank, adapter.data_ptr(), L.RB_I64 if adapter.dtype is torch.int64 else L.RB_I32, _ptr(scale), _ptr(ws), ws_bytes,
             out.data_ptr(), ldo)
    return out


# ------------------------------------------------- attention within segments
_HALVES = (torch.bfloat16, torch.float16)


def _heads_of(t: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """t [T, heads, D] with contiguous columns on 16-byte rows (a copy only where it has none), and its strides."""
    T, heads, D = t.shape
    st, sh, sd = t.stride()
    if (sd != 1 and D > 1) or (D % 8 == 0 and (t.data_ptr() % 16 or (T > 1 and (st % 8 or st <= 0))
                                               or (heads > 1 and (sh % 8 or sh <= 0)))):
        t = t.clone(memory_format=torch.contiguous_format)  # (a contiguous one may start off 16 bytes)
        st, sh = heads * D, D
    return t, st, sh


def _attention_args(name, q, k, v, offsets, k_offsets, causal, prefix, slopes, cap, scale):
    """What both directions check: (device, strided q, k and v, sizes and mask arguments of the entry points)."""
    dev = _device_of(name, q, k, v, offsets, k_offsets, prefix, slopes)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"{name} expects q [Tq, H, D] and k, v [Tk, Hk, D]")
    (Tq, H, D), (Tk, Hk, _) = q.shape, k.shape
    dtype = q.dtype
    if dtype not in _HALVES or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k and v must all be bf16 or all f16")
    if k.shape[2] != D or D == 0 or H == 0 or Hk == 0 or H % Hk:
        raise ValueError(f"k and v must be [Tk, Hk, {D}] with Hk a divisor of {H}, and no dimension of a head empty")
    if k_offsets is None:
        if Tq != Tk:
            raise ValueError("without k_offsets there must be as many keys as queries")
        k_offsets = offsets
    idx = _INDEX.get(offsets.dtype)
    if idx is None or offsets.dim() != 1 or offsets.numel() < 1 or k_offsets.shape != offsets.shape \
            or k_offsets.dtype is not offsets.dtype:
        raise ValueError("offsets (and k_offsets, alike) must be int32 or int64 [segments + 1]")
    S = offsets.numel() - 1
    if prefix is not None:
        if prefix.shape != (S,) or prefix.dtype not in _INDEX:
            raise ValueError(f"prefix must be int32 or int64 [{S}]")
        if prefix.dtype is not offsets.dtype:  # (what int32 cannot hold is more than any segment has)
            prefix = prefix.clamp(0, 2 ** 31 - 1).to(offsets.dtype)
        prefix = prefix.contiguous()
    if slopes is not None:
        if slopes.shape != (H,) or slopes.dtype is not torch.float32:
            raise ValueError(f"slopes must be fp32 [{H}]")
        slopes = slopes.contiguous()
    scale = D ** -0.5 if scale is None else float(scale)
    q, k, v = _heads_of(q), _heads_of(k), _heads_of(v)
    offsets, k_offsets = offsets.contiguous(), k_offsets.contiguous()
    sizes = (_DT[dtype], Tq, Tk, H, Hk, D)
    mask = (offsets, k_offsets, prefix, idx, S, bool(causal), slopes, float(cap), scale)
    return dev, q, k, v, sizes, mask


def segment_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor,
                      k_offsets: Optional[torch.Tensor] = None, *, causal: bool = True,
                      prefix: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None, cap: float = 0.0,
                      scale: Optional[float] = None, want_lse: bool = False):
    """Attention within packed segments (rb_segment_attention): softmax over the keys of a query's own segment.

    q [Tq, H, D], k and v [Tk, Hk, D] bf16/f16 (views of one projection do; Hk divides H), D <= 256; segment s has
    queries offsets[s] .. offsets[s + 1] and keys k_offsets[s] .. (default: the same rows).  Query i of n sees key j of m
    if not `causal`, if j <= i + m - n, or if j < prefix[s].  Scores are scale q.k (default D ** -0.5), with `cap` > 0
    cap tanh(. / cap), with fp32 slopes [H] less slopes[h] |i + m - n - j|.  A query that sees nothing (rows outside
    every segment among them) gets zeros.  Returns (out [Tq, H, D], lse fp32 [H, Tq] or None)."""
    dev, (q, qt, qh), (k, kt, kh), (v, vt, vh), sizes, mask = _attention_args(
        "segment_attention", q, k, v, offsets, k_offsets, causal, prefix, slopes, cap, scale)
    _, Tq, Tk, H, Hk, D = sizes
    off, k_off, prefix, idx, S, causal, slopes, cap, scale = mask
    out = torch.empty((Tq, H, D), dtype=q.dtype, device=dev)
    lse = torch.empty((H, Tq), dtype=torch.float32, device=dev) if want_lse else None
    ws_bytes = _plan_bytes(dev, "rb_segment_attention_workspace_size", Tq, Tk, S, H, Hk, D)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    _call_on(dev, "rb_segment_attention", q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, *sizes,
             off.data_ptr(), k_off.data_ptr(), _ptr(prefix), idx, S, causal, _ptr(slopes), cap, scale, ws.data_ptr(), ws_bytes,
             out.data_ptr(), _ptr(lse))
    return out, lse


def segment_attention_backward(grad: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                               lse: torch.Tensor, offsets: torch.Tensor, k_offsets: Optional[torch.Tensor] = None, *,
                               causal: bool = True, prefix: Optional[torch.Tensor] = None,
                               slopes: Optional[torch.Tensor] = None, cap: float = 0.0, scale: Optional[float] = None):
    """Gradients (q [Tq, H, D], k, v [Tk, Hk, D]) of segment_attention (rb_segment_attention_backward) from that of its
    output and the forward call's inputs, output and lse.  The same bits every time; slopes get no gradient."""
    dev, (q, qt, qh), (k, kt, kh), (v, vt, vh), sizes, mask = _attention_args(
        "segment_attention_backward", q, k, v, offsets, k_offsets, causal, prefix, slopes, cap, scale)
    _device_of("segment_attention_backward", q, grad, out, lse)
    dtype, Tq, Tk, H, Hk, D = sizes
    off, k_off, prefix, idx, S, causal, slopes, cap, scale = mask
    for t in (grad, out):
        if t.shape != (Tq, H, D) or t.dtype is not q.dtype:
            raise ValueError(f"grad and out must be [{Tq}, {H}, {D}] in q's type")
    if lse.shape != (H, Tq) or lse.dtype is not torch.float32 or not lse.is_contiguous():
        raise ValueError(f"lse must be the forward call's fp32 [{H}, {Tq}]")
    grad, gt, gh = _heads_of(grad)
    out = out.contiguous()
    dq = torch.empty((Tq, H, D), dtype=q.dtype, device=dev)
    dk = torch.empty((Tk, Hk, D), dtype=q.dtype, device=dev)
    dv = torch.empty_like(dk)
    ws_bytes = _plan_bytes(dev, "rb_segment_attention_backward_workspace_size", Tq, Tk, S, H, Hk, D)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    _call_on(dev, "rb_segment_attention_backward", grad.data_ptr(), gt, gh, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh,
             v.data_ptr(), vt, vh, out.data_ptr(), lse.data_ptr(), *sizes, off.data_ptr(), k_off.data_ptr(), _ptr(prefix), idx, S,
             causal, _ptr(slopes), cap, scale, ws.data_ptr(), ws_bytes, dq.data_ptr(), dk.data_ptr(), dv.data_ptr())
    return dq, dk, dv


# ------------------------------------------- embedding rows and their gradient
# A kernel wrote into a caller's tensors: autograd's check that what it saved is unchanged has to know.
_written = torch.autograd.graph.increment_version


def embed_rows(table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """scale * table[ids] (rb_embed_rows): table [V, D] fp32/bf16/f16 with contiguous rows, ids int32/int64 of any
    shape, clamped to [0, V - 1].  Returns [*ids.shape, D] in the table's type."""
    dev = _device_of("embed_rows", table, ids)
    if table.dim() != 2 or table.dtype not in _FLOATS or table.shape[1] == 0:
        raise ValueError("embed_rows expects a table [V, D] in fp32, bf16 or f16")
    if ids.dtype not in _INDEX:
        raise ValueError("ids must be int32 or int64")
    V, D = table.shape
    table, ld = _rows_of(table, V, D)
    out = torch.empty((*ids.shape, D), dtype=table.dtype, device=dev)
    ids = ids.contiguous()
    _call_on(dev, "rb_embed_rows", table.data_ptr(), _DT[table.dtype], ld, V, D, ids.data_ptr(), _INDEX[ids.dtype], ids.numel(),
             float(scale), out.data_ptr(), D)
    return out


def _embed_grad_args(name, grad, ids, rows, bags, padding_idx):
    """What both forms of the gradient check: (device, grad rows, their pitch, width, ids, bags, number of bags, padding)."""
    dev = _device_of(name, grad, ids, bags)
    if grad.dim() < 1 or grad.dtype not in _FLOATS or grad.shape[-1] == 0:
        raise ValueError(f"{name} expects grad [..., D] in fp32, bf16 or f16")
    if ids.dtype not in _INDEX:
        raise ValueError("ids must be int32 or int64")
    if rows < 0:
        raise ValueError("the table cannot have a negative number of rows")
    D = grad.shape[-1]
    n_bags = 0
    if bags is None:
        if grad.shape[:-1] != ids.shape:
            raise ValueError(f"grad must be [{', '.join(map(str, ids.shape))}, D]")
    else:
        if ids.dim() != 1 or bags.dim() != 1 or bags.numel() < 1 or bags.dtype not in _INDEX:
            raise ValueError("with bags, ids are [n] and bags int32 or int64 [bags + 1]")
        n_bags = bags.numel() - 1
        if grad.shape != (n_bags, D):
            raise ValueError(f"grad must be [{n_bags}, D], a row a bag")
        bags = bags.to(ids.dtype).contiguous()
    grad, ld = _rows2d(grad, D)
    padding = -1
    if padding_idx is not None:
        if not 0 <= padding_idx < max(rows, 1):
            raise ValueError(f"padding_idx must be in [0, {rows})")
        padding = padding_idx
    return dev, grad, ld, D, ids.contiguous(), bags, n_bags, padding


def embed_rows_backward(grad: torch.Tensor, ids: torch.Tensor, rows: int, *, bags: Optional[torch.Tensor] = None,
                        scale: float = 1.0, padding_idx: Optional[int] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient [rows, D] of embed_rows' table (rb_embed_rows_backward): for each row scale times the sum of grad over the
    ids that name it (clamped as the lookup clamps them), zeros where none does; the same bits every time.

    grad [*ids.shape, D]; with `bags` (offsets [bags + 1] into ids [n]) grad [bags, D], every id taking its bag's row: the
    gradient of sum-pooled bags, ids in no bag taking none.  Ids of padding_idx add nothing.  With `out` [rows, D] (any
    float type) the sums are added to what it holds, rows that no id names being left as they were."""
    dev, grad, ld, D, ids, bags, n_bags, padding = _embed_grad_args("embed_rows_backward", grad, ids, rows, bags, padding_idx)
    given = out is not None
    if not given:
        out = torch.empty((rows, D), dtype=grad.dtype, device=dev)
    else:
        _device_of("embed_rows_backward", grad, out)
        if out.shape != (rows, D) or out.dtype not in _FLOATS or (D > 1 and out.stride(1) != 1) \
                or (rows > 1 and out.stride(0) < D):
            raise ValueError(f"out must be a row-major [{rows}, {D}] tensor in fp32, bf16 or f16")
    n = ids.numel()
    ws_bytes = _plan_bytes(dev, "rb_embed_rows_backward_workspace_size", n, D)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    _call_on(dev, "rb_embed_rows_backward", grad.data_ptr(), _DT[grad.dtype], ld, D, ids.data_ptr(), _INDEX[ids.dtype], n, rows,
             _ptr(bags), n_bags, padding, float(scale), given, ws.data_ptr(), ws_bytes, out.data_ptr(), _DT[out.dtype],
             max(out.stride(0), D))
    if given:
        _written(out)
    return out


def embed_rows_backward_sparse(grad: torch.Tensor, ids: torch.Tensor, rows: int, *, bags: Optional[torch.Tensor] = None,
                               scale: float = 1.0, padding_idx: Optional[int] = None,
                               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """embed_rows_backward of the touched rows alone (rb_embed_rows_backward_sparse).

    Returns (row ids int64 [n], ascending; their gradients [n, D]; count int32 [1] on the device): the first `count`
    entries hold, those behind are left as they were (of fresh tensors: any values).  n is ids.numel(); `out` gives
    both buffers, the gradients' in any float type."""
    name = "embed_rows_backward_sparse"
    dev, grad, ld, D, ids, bags, n_bags, padding = _embed_grad_args(name, grad, ids, rows, bags, padding_idx)
    n = ids.numel()
    given = out is not None
    if not given:
        out = torch.empty((n,), dtype=torch.int64, device=dev), torch.empty((n, D), dtype=grad.dtype, device=dev)
    out_ids, out_rows = out
    _device_of(name, grad, out_ids, out_rows)
    if out_ids.shape != (n,) or out_ids.dtype is not torch.int64 or not out_ids.is_contiguous():
        raise ValueError(f"out's ids must be contiguous int64 [{n}]")
    if out_rows.shape != (n, D) or out_rows.dtype not in _FLOATS or (D > 1 and out_rows.stride(1) != 1) \
            or (n > 1 and out_rows.stride(0) < D):
        raise ValueError(f"out's rows must be a row-major [{n}, {D}] tensor in fp32, bf16 or f16")
    count = torch.empty((1,), dtype=torch.int32, device=dev)
    ws_bytes = _plan_bytes(dev, "rb_embed_rows_backward_workspace_size", n, D)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    _call_on(dev, "rb_embed_rows_backward_sparse", grad.data_ptr(), _DT[grad.dtype], ld, D, ids.data_ptr(), _INDEX[ids.dtype], n,
             rows, _ptr(bags), n_bags, padding, float(scale), ws.data_ptr(), ws_bytes, out_ids.data_ptr(), out_rows.data_ptr(),
             _DT[out_rows.dtype], max(out_rows.stride(0), D), count.data_ptr())
    if given:
        _written((out_ids, out_rows))
    return out_ids, out_rows, count


# ----------------------------------------------- the norm of all gradients
def _dense(t: torch.Tensor) -> bool:
    """Whether t's values fill one run of memory, in whatever order."""
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != at:
            return False
        at *= size
    return True


def _gradients(name: str, grads):
    """(tensors, row counts or None) of a list of gradients, pairs (rows, count) among them."""
    if set(map(type, grads)) <= _PLAIN:
        return grads, None
    tensors, counts = [], {}
    for i, g in enumerate(grads):
        if isinstance(g, torch.Tensor):
            tensors.append(g)
            continue
        rows, count = g
        if rows.dim() != 2 or not rows.is_contiguous() or count.numel() != 1 or count.dtype is not torch.int32:
            raise ValueError(f"{name}: counted rows are a contiguous [n, D] and an int32 [1]")
        counts[i] = count
        tensors.append(rows)
    return tensors, counts


_dtype_of, _T, _PLAIN = operator.attrgetter("dtype"), torch.Tensor, {torch.Tensor, torch.nn.Parameter}


def _clip(name: str, grads, most: float, out, scale: float) -> torch.Tensor:
    # (a call has hundreds of tensors: what is asked of each is asked by map, without Python code per tensor)
    tensors, counts = _gradients(name, grads)
    n = len(tensors)
    if n == 0:
        raise ValueError(f"{name} expects at least one gradient")
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"{name} expects CUDA tensors")
    index = dev.index
    if set(map(_T.get_device, tensors)) != {index} or (counts and any(c.device != dev for c in counts.values())):
        raise RuntimeError(f"{name}: tensors on different devices")
    dtypes = list(map(_dtype_of, tensors))
    if not set(dtypes) <= _GRAD_TYPES.keys():
        raise ValueError("gradients must be fp32, bf16 or f16")
    clip = most >= 0.0
    back = []  # (a copy, where it goes): gradients whose values lie apart
    whole = all(map(_T.is_contiguous, tensors))
    if not whole:
        for i, t in enumerate(tensors):
            if not _dense(t):
                tensors[i] = t.contiguous()
                if clip and out is None:
                    back.append((tensors[i], t))
    sizes = array("q", map(_T.numel, tensors))
    ptrs = to = array("q", map(_T.data_ptr, tensors))
    if not clip:
        to = None
    elif out is not None:
        if len(out) != n or set(map(_T.get_device, out)) != {index} or list(map(_dtype_of, out)) != dtypes or \
                array("q", map(_T.numel, out)) != sizes or \
                not (whole and all(map(_T.is_contiguous, out)) or
                     all(o.stride() == t.stride() and _dense(o) for o, t in zip(out, tensors))):
            raise ValueError("out's tensors must be as the gradients, their values in one run of memory")
        to = array("q", map(_T.data_ptr, out))
    if clip and len(set(to)) < n and len({a for a, m in zip(to, sizes) if m}) < sum(1 for m in sizes if m):
        raise ValueError(f"{name}: a tensor to be clipped was given twice")
    types = array("i", map(_GRAD_TYPES.__getitem__, dtypes))
    counted = widths = None
    if counts:
        counted, widths = array("q", bytes(8 * n)), array("q", bytes(8 * n))
        for i, c in counts.items():
            counted[i], widths[i] = c.data_ptr(), max(tensors[i].shape[1], 1)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws_bytes = _plan_bytes(dev, "rb_grad_norm_workspace_size", n)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    lists = [None if a is None else a.buffer_info()[0] for a in (ptrs, to, sizes, types, counted, widths)]
    _call_on(dev, "rb_clip_grads", *lists, n, float(scale), float(most), ws.data_ptr(), ws_bytes, norm.data_ptr())
    if clip:
        _written(tensors if out is None else out)
    for copy, t in back:
        t.copy_(copy)
    return norm


_GRAD_TYPES = {t: _DT[t] for t in _FLOATS}


def grad_norm(grads, *, scale: float = 1.0) -> torch.Tensor:
    """scale times the 2-norm of all values of `grads` together, fp32 [] on the device (rb_clip_grads without clipping).

    Each gradient is a tensor (fp32, bf16, f16; any shape), or a pair (rows [n, D], count int32 [1]) of which the first
    `count` rows count (what embed_rows_backward_sparse returns)."""
    return _clip("grad_norm", list(grads), -1.0, None, scale)


def clip_grads(grads, max_norm: float, *, out=None, scale: float = 1.0) -> torch.Tensor:
    """Clip gradients by their norm together (rb_clip_grads): with norm = grad_norm(grads, scale=scale), each gradient
    becomes scale * g * min(1, max_norm / (norm + 1e-6)), in place or in the tensors `out` (laid out as the gradients).
    Returns the norm, which nothing waits for.  A norm of NaN makes all of them NaN, an infinite one zeros (and NaN where
    they are infinite).  Tensors must not share memory."""
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative")
    return _clip("clip_grads", list(grads), max_norm, None if out is None else list(out), scale)


def device_error(reset: bool = False) -> int:
    return L.device_error(reset)


def selftest_wait_timeout(budget_ns: int, device=None) -> None:
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        L.call("rb_selftest_wait_timeout", int(budget_ns), _stream(dev))
