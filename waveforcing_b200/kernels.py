"""torch-facing wrappers over the libwfk C ABI.

Each wrapper validates dtype/device/layout, launches on the caller's current
CUDA stream and raises on any error.  There is no CPU or library fallback:
CPU tensors or a missing libwfk.so raise.
"""

from __future__ import annotations

import ctypes as C
import math
import struct

import torch

from waveforcing_b200 import _lib as L

# Number of libwfk kernel launches issued through these wrappers (reported by
# bench.py as gpu_launches for its timed region).
LAUNCHES = [0]


def _stream() -> int:
    LAUNCHES[0] += 1
    return torch.cuda.current_stream().cuda_stream


def _check(cond: bool, msg: str) -> None:
    """Shape/dtype validation the C ABI cannot do: it sees pointers, not sizes,
    so a mis-shaped output or side tensor would be read or written out of
    bounds.  Runs before the device check."""
    if not cond:
        raise ValueError(msg)


def _need_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("waveforcing_b200 kernels need CUDA tensors (no CPU path exists)")


def _strides_bthd(t: torch.Tensor):
    """[B, L, H, D] or [L, H, D] -> (batch, L, H, D, {batch, token, head} strides)."""
    if t.dim() == 3:
        Lt, H, D = t.shape
        return 1, Lt, H, D, (t.stride(0) * Lt, t.stride(0), t.stride(1))
    if t.dim() == 4:
        B, Lt, H, D = t.shape
        return B, Lt, H, D, (t.stride(0), t.stride(1), t.stride(2))
    raise ValueError(f"expected [B,L,H,D] or [L,H,D], got {tuple(t.shape)}")


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T * scale) v on the tcgen05 kernel; NHD bf16, head_dim 128."""
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise TypeError("attention: q, k, v must be bfloat16")
    for t in (q, k, v):
        if t.stride(-1) != 1:
            raise ValueError("attention: last dim must be contiguous")
    B, Lq, H, D, qs = _strides_bthd(q)
    Bk, Lk, Hk, Dk, ks = _strides_bthd(k)
    Bv, Lv, Hv, Dv, vs = _strides_bthd(v)
    if (Bk, Hk, Dk) != (B, H, D) or (Bv, Lv, Hv, Dv) != (B, Lk, H, D):
        raise ValueError(f"attention: shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _check(out.shape == q.shape and out.dtype == torch.bfloat16 and out.device == q.device and out.stride(-1) == 1,
           "attention: out must be bf16 with q's shape and device and a contiguous last dim")
    _need_cuda(q, k, v, out)
    _, _, _, _, os_ = _strides_bthd(out)
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    L.check(
        L.lib().wf_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, Lq, Lk, H, D,
                            L.i64_array(qs), L.i64_array(ks), L.i64_array(vs), L.i64_array(os_),
                            L.WF_DTYPE_BF16, None, None, L.WF_SCALE_NONE, scale, _stream()),
        "wf_attn_fwd",
    )
    return out


def attention_fp8(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor | None,
                  v_scale: torch.Tensor | None, scale_mode: int = L.WF_SCALE_TOKEN, softmax_scale: float | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention over FP8 K/V pages: q bf16 [B, Lq, H, 128]; k_codes/v_codes
    uint8 e4m3 codes [B, Lk, H, 128]; scales f32 per token row [B, Lk]
    (WF_SCALE_TOKEN), one per tensor [1] (WF_SCALE_TENSOR) or none.  The
    kernel expands the codes to f16 products code * scale in shared memory and
    runs both contractions on f16 operands (|q| and |k|, |v| below 65504)."""
    if q.dtype != torch.bfloat16 or k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8:
        raise TypeError("attention_fp8: q must be bfloat16, k/v uint8 e4m3 codes")
    for t in (q, k_codes, v_codes):
        if t.stride(-1) != 1:
            raise ValueError("attention_fp8: last dim must be contiguous")
    B, Lq, H, D, qs = _strides_bthd(q)
    Bk, Lk, Hk, Dk, ks = _strides_bthd(k_codes)
    Bv, Lv, Hv, Dv, vs = _strides_bthd(v_codes)
    if (Bk, Hk, Dk) != (B, H, D) or (Bv, Lv, Hv, Dv) != (B, Lk, H, D):
        raise ValueError(f"attention_fp8: shape mismatch q{tuple(q.shape)} k{tuple(k_codes.shape)} "
                         f"v{tuple(v_codes.shape)}")
    need = {L.WF_SCALE_TOKEN: B * Lk, L.WF_SCALE_TENSOR: 1, L.WF_SCALE_NONE: 0}.get(scale_mode)
    _check(need is not None, "attention_fp8: unknown scale_mode")
    if need:
        _check(all(t is not None and t.dtype == torch.float32 and t.is_contiguous() and t.numel() >= need
                   for t in (k_scale, v_scale)),
               "attention_fp8: k_scale/v_scale must be contiguous f32 with B*Lk (token) or 1 (tensor) elements")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _check(out.shape == q.shape and out.dtype == torch.bfloat16 and out.stride(-1) == 1,
           "attention_fp8: out must be bf16 with q's shape and a contiguous last dim")
    _need_cuda(q, k_codes, v_codes, out)
    _, _, _, _, os_ = _strides_bthd(out)
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    L.check(
        L.lib().wf_attn_fwd(q.data_ptr(), k_codes.data_ptr(), v_codes.data_ptr(), out.data_ptr(), B, Lq, Lk, H, D,
                            L.i64_array(qs), L.i64_array(ks), L.i64_array(vs), L.i64_array(os_),
                            L.WF_DTYPE_E4M3, k_scale.data_ptr() if need else None,
                            v_scale.data_ptr() if need else None, scale_mode, scale, _stream()),
        "wf_attn_fwd(e4m3)",
    )
    return out


def _as_rows(x: torch.Tensor):
    """View x as [rows, cols] with a row stride (last dim contiguous)."""
    if x.dim() == 1:
        return 1, x.shape[0], x.shape[0]
    cols = x.shape[-1]
    x2 = x.reshape(-1, cols) if not x.is_contiguous() else x.view(-1, cols)
    return x2.shape[0], cols, x2.stride(0)


def kv_quant(x: torch.Tensor, mode: int = L.WF_SCALE_TOKEN, codes: torch.Tensor | None = None,
             scales: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """bf16 [rows, cols] -> (u8 codes [rows, cols], f32 scales [rows] or [1])."""
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.stride(-1) != 1:
        raise ValueError("kv_quant: x must be a 2-D bf16 matrix with contiguous rows")
    rows, cols = x.shape
    n_scales = rows if mode == L.WF_SCALE_TOKEN else 1
    if codes is not None:
        _check(codes.dtype == torch.uint8 and codes.is_contiguous() and codes.numel() == rows * cols,
               "kv_quant: codes must be a contiguous uint8 tensor of rows * cols elements")
    if scales is not None and mode != L.WF_SCALE_NONE:
        _check(scales.dtype == torch.float32 and scales.is_contiguous() and scales.numel() >= n_scales,
               "kv_quant: scales must be contiguous f32 with one element per row (token) or one (tensor)")
    if workspace is not None:
        _check(workspace.dtype == torch.int32 and workspace.numel() >= 1,
               "kv_quant: workspace must be an int32 tensor of at least one element")
    _need_cuda(x)
    if codes is None:
        codes = torch.empty((rows, cols), dtype=torch.uint8, device=x.device)
    if scales is None and mode != L.WF_SCALE_NONE:
        scales = torch.empty((n_scales,), dtype=torch.float32, device=x.device)
    ws = 0
    if mode == L.WF_SCALE_TENSOR:
        if workspace is None:
            workspace = torch.empty((1,), dtype=torch.int32, device=x.device)
        ws = workspace.data_ptr()
    L.check(L.lib().wf_kv_quant(x.data_ptr(), codes.data_ptr(), scales.data_ptr() if scales is not None else None,
                                rows, cols, x.stride(0), mode, ws, _stream()), "wf_kv_quant")
    return codes, scales


def kv_dequant(codes: torch.Tensor, scales: torch.Tensor | None, mode: int = L.WF_SCALE_TOKEN,
               out: torch.Tensor | None = None) -> torch.Tensor:
    if codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.is_contiguous():
        raise ValueError("kv_dequant: codes must be a contiguous 2-D uint8 matrix")
    rows, cols = codes.shape
    if mode != L.WF_SCALE_NONE:
        _check(scales is not None and scales.dtype == torch.float32
               and scales.numel() >= (rows if mode == L.WF_SCALE_TOKEN else 1),
               "kv_dequant: f32 scales needed, one per row (token) or one (tensor)")
    if out is not None:
        _check(out.dim() == 2 and tuple(out.shape) == (rows, cols) and out.dtype == torch.bfloat16
               and out.stride(-1) == 1, "kv_dequant: out must be bf16 [rows, cols] with contiguous rows")
    _need_cuda(codes)
    if out is None:
        out = torch.empty((rows, cols), dtype=torch.bfloat16, device=codes.device)
    sp = scales.data_ptr() if scales is not None else 0
    L.check(L.lib().wf_kv_dequant(codes.data_ptr(), sp, out.data_ptr(), rows, cols, out.stride(0), mode, _stream()),
            "wf_kv_dequant")
    return out


def kv_quant_publish(k: torch.Tensor, v: torch.Tensor, dst_codes_k, dst_codes_v, dst_scales_k, dst_scales_v) -> None:
    """Per-token quantise K and V [rows, cols] and write codes/scales to every
    destination (device pointers as ints, local or peer)."""
    _check(k.dim() == 2 and v.shape == k.shape and k.dtype == v.dtype == torch.bfloat16,
           "kv_quant_publish: k and v must be bf16 matrices of one shape")
    n = len(dst_codes_k)
    _check(n >= 1 and len(dst_codes_v) == len(dst_scales_k) == len(dst_scales_v) == n,
           "kv_quant_publish: one code and one scale destination per K and V, same count")
    _need_cuda(k, v)
    rows, cols = k.shape
    L.check(L.lib().wf_kv_quant_publish(k.data_ptr(), v.data_ptr(), rows, cols, k.stride(0), v.stride(0),
                                        L.ptr_array(dst_codes_k), L.ptr_array(dst_codes_v),
                                        L.ptr_array(dst_scales_k), L.ptr_array(dst_scales_v), n, _stream()),
            "wf_kv_quant_publish")


def weight_quant(w: torch.Tensor, qtype: int = L.WF_DTYPE_E4M3):
    """bf16 [N, K] -> (codes [N, K] uint8/int8 storage, f32 scales [N])."""
    _check(w.dim() == 2 and w.dtype == torch.bfloat16, "weight_quant: w must be a bf16 [N, K] matrix")
    _need_cuda(w)
    w = w.contiguous()
    N, K = w.shape
    wq = torch.empty((N, K), dtype=torch.uint8, device=w.device)
    ws = torch.empty((N,), dtype=torch.float32, device=w.device)
    L.check(L.lib().wf_weight_quant(w.data_ptr(), wq.data_ptr(), ws.data_ptr(), N, K, qtype, _stream()),
            "wf_weight_quant")
    return wq, ws


def act_quant(x: torch.Tensor, qtype: int = L.WF_DTYPE_E4M3, xq: torch.Tensor | None = None,
              xs: torch.Tensor | None = None, activation: int = L.WF_ACT_NONE):
    """Per-token activation quantisation of x [M, K] bf16; activation
    WF_ACT_GELU_TANH quantises bf16(GELU_tanh(x)) instead."""
    _check(x.dim() == 2 and x.dtype == torch.bfloat16 and x.stride(-1) == 1,
           "act_quant: x must be a bf16 [M, K] matrix with contiguous rows")
    M, K = x.shape
    _check(xq is None or tuple(xq.shape) == (M, K), "act_quant: xq must be [M, K]")
    _check(xs is None or (xs.dtype == torch.float32 and xs.numel() >= M), "act_quant: xs must hold M f32 scales")
    _need_cuda(x)
    if xq is None:
        xq = torch.empty((M, K), dtype=torch.uint8, device=x.device)
    if xs is None:
        xs = torch.empty((M,), dtype=torch.float32, device=x.device)
    L.check(L.lib().wf_act_quant_act(x.data_ptr(), xq.data_ptr(), xs.data_ptr(), M, K, x.stride(0), qtype,
                                     activation, _stream()), "wf_act_quant_act")
    return xq, xs


def gemm_w8a8(xq, xs, wq, ws, bias=None, qtype: int = L.WF_DTYPE_E4M3, scale_mode: int = L.WF_SCALE_TOKEN,
              out: torch.Tensor | None = None, activation: int = L.WF_ACT_NONE) -> torch.Tensor:
    """y = (xq wq^T) * xs * ws + bias in bf16; activation WF_ACT_GELU_TANH applies
    GELU(tanh) to the bf16-rounded result in the same kernel."""
    _check(xq.dim() == 2 and wq.dim() == 2 and xq.shape[1] == wq.shape[1],
           "gemm_w8a8: xq [M, K] and wq [N, K] must share K")
    M, K = xq.shape
    N = wq.shape[0]
    per_token = scale_mode == L.WF_SCALE_TOKEN
    _check(xs.dtype == ws.dtype == torch.float32 and xs.numel() >= (M if per_token else 1)
           and ws.numel() >= (N if per_token else 1),
           "gemm_w8a8: f32 scales needed, x_scale per row and w_scale per channel (one each per tensor)")
    _check(bias is None or bias.numel() == N, "gemm_w8a8: bias must have N elements")
    _check(out is None or (tuple(out.shape) == (M, N) and out.dtype == torch.bfloat16 and out.stride(-1) == 1),
           "gemm_w8a8: out must be bf16 [M, N] with contiguous rows")
    _need_cuda(xq, wq)
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=xq.device)
    bp = bias.data_ptr() if bias is not None else 0
    L.check(L.lib().wf_gemm_w8a8_act(xq.data_ptr(), xs.data_ptr(), wq.data_ptr(), ws.data_ptr(), bp, out.data_ptr(),
                                     M, N, K, out.stride(0), qtype, scale_mode, activation, _stream()),
            "wf_gemm_w8a8_act")
    return out


def kv_assemble(segments, cols: int, head_dim: int) -> None:
    """One launch that fills K/V context rows from a list of segments
    (kind, src, aux0, aux1, dst, rows, src_row_stride, dst_row_stride), with
    kind WF_SEG_COPY / WF_SEG_ROPE / WF_SEG_DEQUANT, pointers as ints (aux as 0
    when unused) and strides in elements of the source / bf16 destination."""
    n = len(segments)
    arr = (L.KvSegment * max(1, n))()
    for i, (kind, src, a0, a1, dst, rows, ss, ds) in enumerate(segments):
        arr[i] = L.KvSegment(kind, 0, src, a0 or None, a1 or None, dst, rows, ss, ds)
    L.check(L.lib().wf_kv_assemble(arr, n, cols, head_dim, _stream()), "wf_kv_assemble")


def rope_apply(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, out: torch.Tensor | None = None):
    """Interleaved RoPE on bf16 [L, H, D] with f32 cos/sin [L, D/2]."""
    if x.dim() == 4:
        x = x[0]
    Lt, H, D = x.shape
    _check(x.dtype == torch.bfloat16 and x.stride(2) == 1 and x.stride(1) == D,
           "rope_apply: x must be bf16 [L, H, D] with contiguous heads (token stride is free)")
    for tab in (cos, sin):
        _check(tab.dtype == torch.float32 and tab.dim() == 2 and tab.shape[0] >= Lt and tab.shape[1] == D // 2
               and tab.is_contiguous(), "rope_apply: cos/sin must be contiguous f32 [>= L, D/2]")
    _check(out is None or (out.shape == x.shape and out.dtype == x.dtype and out.stride(2) == 1
                           and out.stride(1) == D), "rope_apply: out must match x, with contiguous heads")
    _need_cuda(x, cos, sin)
    if out is None:
        out = torch.empty_like(x)
    L.check(L.lib().wf_rope_apply(x.data_ptr(), out.data_ptr(), cos.data_ptr(), sin.data_ptr(), Lt, H, D,
                                  x.stride(0), out.stride(0), _stream()), "wf_rope_apply")
    return out


# ------------------------------------------------------ fused Wan-block rows
def ln_modulate(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, rows_per_stage: int, eps: float,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """out = LN(x) * (1 + scale[s]) + shift[s]; x bf16 [rows, dim], shift/scale f32 [S, dim] row-strided."""
    _check(x.dim() == 2 and x.dtype == torch.bfloat16, "ln_modulate: x must be a bf16 [rows, dim] matrix")
    rows, dim = x.shape
    for t in (shift, scale):
        _check(t.dtype == torch.float32 and t.dim() == 2 and t.shape[1] == dim and t.stride(1) == 1
               and t.shape[0] * rows_per_stage >= rows, "ln_modulate: shift/scale must be f32 [stages, dim]")
    _check(shift.stride(0) == scale.stride(0), "ln_modulate: shift and scale must share their row stride")
    _check(out is None or (out.shape == x.shape and out.dtype == torch.bfloat16), "ln_modulate: out must match x")
    _need_cuda(x)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    L.check(L.lib().wf_ln_modulate(x.data_ptr(), x.stride(0), shift.data_ptr(), scale.data_ptr(), shift.stride(0),
                                   out.data_ptr(), out.stride(0), rows, dim, rows_per_stage, eps, _stream()),
            "wf_ln_modulate")
    return out


def ln_modulate_quant(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, rows_per_stage: int, eps: float,
                      qtype: int = L.WF_DTYPE_E4M3):
    """ln_modulate followed by the per-token W8A8 activation quantiser, in one
    kernel: returns (codes uint8 [rows, dim], scales f32 [rows]), equal to
    act_quant(ln_modulate(x)) without the bf16 output being written."""
    _check(x.dim() == 2 and x.dtype == torch.bfloat16, "ln_modulate_quant: x must be a bf16 [rows, dim] matrix")
    rows, dim = x.shape
    for t in (shift, scale):
        _check(t.dtype == torch.float32 and t.dim() == 2 and t.shape[1] == dim and t.stride(1) == 1
               and t.shape[0] * rows_per_stage >= rows, "ln_modulate_quant: shift/scale must be f32 [stages, dim]")
    _check(shift.stride(0) == scale.stride(0), "ln_modulate_quant: shift and scale must share their row stride")
    _need_cuda(x)
    xq = torch.empty((rows, dim), device=x.device, dtype=torch.uint8)
    xs = torch.empty((rows,), device=x.device, dtype=torch.float32)
    L.check(L.lib().wf_ln_modulate_quant(x.data_ptr(), x.stride(0), shift.data_ptr(), scale.data_ptr(),
                                         shift.stride(0), xq.data_ptr(), xs.data_ptr(), rows, dim, rows_per_stage,
                                         eps, qtype, _stream()), "wf_ln_modulate_quant")
    return xq, xs


def gate_residual(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor, rows_per_stage: int) -> torch.Tensor:
    """x += y * gate[s] in place (f32 math, bf16 storage)."""
    _check(x.dim() == 2 and y.shape == x.shape and x.dtype == y.dtype == torch.bfloat16,
           "gate_residual: x and y must be bf16 matrices of one shape")
    rows, dim = x.shape
    _check(gate.dtype == torch.float32 and gate.shape[-1] == dim and gate.stride(-1) == 1
           and (gate.dim() == 1 or (gate.dim() == 2 and gate.shape[0] * rows_per_stage >= rows)),
           "gate_residual: gate must be f32 [dim] or [stages, dim]")
    _need_cuda(x, y)
    gs = gate.stride(0) if gate.dim() == 2 else 0
    L.check(L.lib().wf_gate_residual(x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), gate.data_ptr(), gs,
                                     rows, dim, rows_per_stage, _stream()), "wf_gate_residual")
    return x


def gate_residual_then(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor, gate_rows_per_stage: int,
                       shift: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                       mod_rows_per_stage: int = 1, eps: float = 1e-6, quant: bool = False,
                       qtype: int = L.WF_DTYPE_E4M3):
    """x += y * gate[s] in place, then from the new rows without reading them
    back: with shift/scale, LN-modulate to a new bf16 [rows, dim] (or, with
    ``quant``, its per-token W8A8 codes and scales); without, the per-token
    quantisation of x itself (``quant`` implied).  Returns the bf16 output or
    (codes uint8 [rows, dim], scales f32 [rows])."""
    _check(x.dim() == 2 and y.shape == x.shape and x.dtype == y.dtype == torch.bfloat16,
           "gate_residual_then: x and y must be bf16 matrices of one shape")
    rows, dim = x.shape
    _check(gate.dtype == torch.float32 and gate.shape[-1] == dim and gate.stride(-1) == 1
           and (gate.dim() == 1 or (gate.dim() == 2 and gate.shape[0] * gate_rows_per_stage >= rows)),
           "gate_residual_then: gate must be f32 [dim] or [stages, dim]")
    mod = shift is not None or scale is not None
    if mod:
        for t in (shift, scale):
            _check(t is not None and t.dtype == torch.float32 and t.dim() == 2 and t.shape[1] == dim
                   and t.stride(1) == 1 and t.shape[0] * mod_rows_per_stage >= rows,
                   "gate_residual_then: shift/scale must be f32 [stages, dim]")
        _check(shift.stride(0) == scale.stride(0), "gate_residual_then: shift and scale must share their row stride")
    _need_cuda(x, y)
    gs = gate.stride(0) if gate.dim() == 2 else 0
    quant = quant or not mod
    out = xq = xs = None
    if quant:
        xq = torch.empty((rows, dim), device=x.device, dtype=torch.uint8)
        xs = torch.empty((rows,), device=x.device, dtype=torch.float32)
    else:
        out = torch.empty((rows, dim), device=x.device, dtype=torch.bfloat16)
    L.check(L.lib().wf_gate_residual_then(
        x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), gate.data_ptr(), gs, gate_rows_per_stage,
        shift.data_ptr() if mod else None, scale.data_ptr() if mod else None, shift.stride(0) if mod else 0,
        mod_rows_per_stage, eps, out.data_ptr() if out is not None else None, dim,
        xq.data_ptr() if quant else None, xs.data_ptr() if quant else None, qtype, rows, dim, _stream()),
        "wf_gate_residual_then")
    return (xq, xs) if quant else out


def channel_rmsnorm(x: torch.Tensor, gamma: torch.Tensor, silu: bool, eps: float = 1e-12,
                    out: torch.Tensor | None = None) -> torch.Tensor:  # out: any contiguous bf16 of x's shape
    """x / max(||x||, eps) * sqrt(C) * gamma over the LAST dimension of a
    contiguous bf16 tensor (the channel rows of channels-last activations),
    then SiLU when ``silu``; ``out`` may be x itself."""
    _check(x.dtype == torch.bfloat16 and x.is_contiguous(), "channel_rmsnorm: x must be contiguous bf16")
    C = x.shape[-1]
    _check(gamma.dtype == torch.bfloat16 and gamma.numel() == C and gamma.is_contiguous(),
           "channel_rmsnorm: gamma must be contiguous bf16 [C]")
    _check(out is None or (out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous()),
           "channel_rmsnorm: out must match x")
    _need_cuda(x)
    if out is None:
        out = torch.empty_like(x)
    L.check(L.lib().wf_channel_rmsnorm(x.data_ptr(), out.data_ptr(), x.numel() // C, C, gamma.data_ptr(), eps,
                                       1 if silu else 0, _stream()), "wf_channel_rmsnorm")
    return out


def channel_bias_add(x: torch.Tensor, bias: torch.Tensor, res: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """x + bias (over the channel dim 1) [+ res] for channels-last bf16 x of 4 or
    5 dims; out may be x.  Returns a tensor in x's layout."""
    cl = torch.channels_last_3d if x.dim() == 5 else torch.channels_last
    _check(x.dtype == torch.bfloat16 and x.dim() in (4, 5) and x.is_contiguous(memory_format=cl),
           "channel_bias_add: x must be channels-last bf16 of 4 or 5 dims")
    C = x.shape[1]
    _check(bias.dtype == torch.bfloat16 and bias.numel() == C and bias.is_contiguous(),
           "channel_bias_add: bias must be contiguous bf16 [C]")
    _check(res is None or (res.shape == x.shape and res.dtype == x.dtype and res.is_contiguous(memory_format=cl)),
           "channel_bias_add: res must match x (channels-last)")
    _need_cuda(x)
    if out is None:
        out = torch.empty_like(x, memory_format=cl)
    L.check(L.lib().wf_channel_bias_add(x.data_ptr(), bias.data_ptr(), res.data_ptr() if res is not None else None,
                                        out.data_ptr(), x.numel() // C, C, _stream()), "wf_channel_bias_add")
    return out


def upsample2x_nearest(f: torch.Tensor) -> torch.Tensor:
    """Nearest x2 in H and W of channels-last bf16 images [N, C, H, W]."""
    _check(f.dtype == torch.bfloat16 and f.dim() == 4 and f.is_contiguous(memory_format=torch.channels_last),
           "upsample2x_nearest: f must be channels-last bf16 [N, C, H, W]")
    n, c, h, w = f.shape
    _need_cuda(f)
    out = torch.empty((n, c, 2 * h, 2 * w), device=f.device, dtype=f.dtype, memory_format=torch.channels_last)
    L.check(L.lib().wf_upsample2x_nearest(f.data_ptr(), out.data_ptr(), n, h, w, c, _stream()),
            "wf_upsample2x_nearest")
    return out


def interleave_time2(y: torch.Tensor) -> torch.Tensor:
    """[b, 2C, T, H, W] channels-last bf16 -> [b, C, 2T, H, W] channels-last:
    frame 2i from channels [0, C) of frame i, frame 2i + 1 from [C, 2C)."""
    _check(y.dim() == 5 and y.dtype == torch.bfloat16 and y.is_contiguous(memory_format=torch.channels_last_3d)
           and y.shape[1] % 2 == 0, "interleave_time2: y must be channels-last bf16 [b, 2C, T, H, W]")
    b, c2, t, h, w = y.shape
    _need_cuda(y)
    out = torch.empty((b, c2 // 2, 2 * t, h, w), device=y.device, dtype=y.dtype,
                      memory_format=torch.channels_last_3d)
    L.check(L.lib().wf_interleave_time2(y.data_ptr(), out.data_ptr(), b * t, h * w, c2 // 2, _stream()),
            "wf_interleave_time2")
    return out


def qk_norm_rope(qkv: torch.Tensor, dim: int, wq: torch.Tensor, wk: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, head_dim: int, rows_per_stage: int, eps: float, want_unroped: bool = True):
    """Fused RMSNorm(q), RMSNorm(k) + RoPE from the fused QKV GEMM output.
    Returns (roped q, roped k, normalised un-roped k or None), each [rows, dim]."""
    _check(qkv.dim() == 2 and qkv.dtype == torch.bfloat16 and qkv.shape[1] >= 3 * dim,
           "qk_norm_rope: qkv must be a bf16 [rows, >= 3*dim] matrix")
    rows = qkv.shape[0]
    _check(all(w.numel() == dim and w.dtype == torch.bfloat16 and w.is_contiguous() for w in (wq, wk)),
           "qk_norm_rope: norm weights must be contiguous bf16 with dim elements")
    for tab in (cos, sin):
        _check(tab.dtype == torch.float32 and tab.dim() == 2 and tab.shape[0] >= rows
               and tab.shape[1] == head_dim // 2 and tab.is_contiguous(),
               "qk_norm_rope: cos/sin must be contiguous f32 [>= rows, head_dim/2]")
    _need_cuda(qkv)
    q = torch.empty((rows, dim), device=qkv.device, dtype=torch.bfloat16)
    k = torch.empty_like(q)
    ku = torch.empty_like(q) if want_unroped else None
    L.check(L.lib().wf_qk_norm_rope(qkv.data_ptr(), qkv.stride(0), wq.data_ptr(), wk.data_ptr(), cos.data_ptr(),
                                    sin.data_ptr(), head_dim, q.data_ptr(), k.data_ptr(),
                                    ku.data_ptr() if ku is not None else None, rows, dim, rows_per_stage, eps,
                                    _stream()), "wf_qk_norm_rope")
    return q, k, ku


def qk_norm_rope_publish(qkv: torch.Tensor, dim: int, wq: torch.Tensor, wk: torch.Tensor, cos: torch.Tensor,
                         sin: torch.Tensor, head_dim: int, rows_per_stage: int, eps: float, publish,
                         want_unroped: bool = True):
    """qk_norm_rope plus the per-token FP8 publish of every stage's roped K and
    V (wf_qk_norm_rope_publish).  ``publish[s]`` lists stage s's destination
    slots as (codes_k, codes_v, scales_k, scales_v) device pointers (ints),
    each slot [rows_per_stage, dim] codes and [rows_per_stage] f32 scales."""
    _check(qkv.dim() == 2 and qkv.dtype == torch.bfloat16 and qkv.shape[1] >= 3 * dim,
           "qk_norm_rope_publish: qkv must be a bf16 [rows, >= 3*dim] matrix")
    rows = qkv.shape[0]
    _check(all(w.numel() == dim and w.dtype == torch.bfloat16 and w.is_contiguous() for w in (wq, wk)),
           "qk_norm_rope_publish: norm weights must be contiguous bf16 with dim elements")
    for tab in (cos, sin):
        _check(tab.dtype == torch.float32 and tab.dim() == 2 and tab.shape[0] >= rows
               and tab.shape[1] == head_dim // 2 and tab.is_contiguous(),
               "qk_norm_rope_publish: cos/sin must be contiguous f32 [>= rows, head_dim/2]")
    n_stages = len(publish)
    _check(n_stages <= L.PUBLISH_MAX_STAGES and n_stages * rows_per_stage >= rows
           and all(len(p) <= L.PUBLISH_MAX_DST for p in publish),
           "qk_norm_rope_publish: one destination list per stage, at most 8 stages of 8 destinations")
    _need_cuda(qkv)
    dsts = (L.KvPublishDst * max(1, n_stages * L.PUBLISH_MAX_DST))()
    counts = (C.c_int32 * max(1, n_stages))()
    for s, lst in enumerate(publish):
        counts[s] = len(lst)
        for d, (ck, cv, sk, sv) in enumerate(lst):
            dsts[s * L.PUBLISH_MAX_DST + d] = L.KvPublishDst(int(ck), int(cv), int(sk), int(sv))
    q = torch.empty((rows, dim), device=qkv.device, dtype=torch.bfloat16)
    k = torch.empty_like(q)
    ku = torch.empty_like(q) if want_unroped else None
    L.check(L.lib().wf_qk_norm_rope_publish(qkv.data_ptr(), qkv.stride(0), wq.data_ptr(), wk.data_ptr(),
                                            cos.data_ptr(), sin.data_ptr(), head_dim, q.data_ptr(), k.data_ptr(),
                                            ku.data_ptr() if ku is not None else None, rows, dim, rows_per_stage,
                                            eps, dsts, counts, n_stages, _stream()), "wf_qk_norm_rope_publish")
    return q, k, ku


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    _check(x.dim() == 2 and x.dtype == torch.bfloat16 and w.numel() == x.shape[1] and w.dtype == torch.bfloat16
           and w.is_contiguous(), "rms_norm: x must be bf16 [rows, dim] and w contiguous bf16 with dim elements")
    _need_cuda(x)
    rows, dim = x.shape
    out = torch.empty((rows, dim), device=x.device, dtype=torch.bfloat16)
    L.check(L.lib().wf_rms_norm(x.data_ptr(), x.stride(0), w.data_ptr(), out.data_ptr(), out.stride(0), rows, dim,
                                eps, _stream()), "wf_rms_norm")
    return out


# ------------------------------------------------- paged K/V cache, cross attention
# These calls are issued per layer and token, so their arguments are packed into
# bytes (struct) rather than built as ctypes objects: 6 us a call instead of 12.
_PACK_PAGES = struct.Struct("4Qq4i10q").pack  # wf_kv_pages
_PACK_BATCH = struct.Struct("Qq2Q2iq").pack   # wf_kv_batch
_PACK2, _PACK3 = struct.Struct("2q").pack, struct.Struct("3q").pack


_SCALE = 1.0 / math.sqrt(128)
_I32 = 2**31 - 1


def _st2(t: torch.Tensor) -> tuple:
    """The first two strides; a dim of one element, whose stride torch leaves open, gets 16."""
    s, n = t.stride(), t.shape
    return (s[0] if n[0] != 1 else 16, s[1] if n[1] != 1 else 16)


def _st3(t: torch.Tensor) -> tuple:
    s, n = t.stride(), t.shape
    return (s[0] if n[0] != 1 else 16, s[1] if n[1] != 1 else 16, s[2] if n[2] != 1 else 16)


_PAGE_DTYPES = {torch.bfloat16: L.WF_DTYPE_BF16, torch.uint8: L.WF_DTYPE_E4M3, torch.int8: L.WF_DTYPE_S8}


class KVPages:
    """K and V pages of one layer: ``k``, ``v`` [pages, kv_heads, page_size, 128]
    as bf16 rows, e4m3 codes (uint8) or signed 8-bit codes (int8), the 8-bit
    forms with f32 ``k_scale``, ``v_scale`` [pages, kv_heads, page_size] (a row's
    value is code * scale).  Strides are free (multiples of 16 bytes, the 128
    elements of a row and the scales of a page contiguous, nothing broadcast), so
    pages stored token-major are passed as a transposed view."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "kv_dtype")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> None:
        dtype, shape, d = k.dtype, k.shape, k.get_device()
        if not (dtype in _PAGE_DTYPES and v.dtype is dtype):
            raise ValueError("KVPages: k and v must both be bf16, uint8 (e4m3) or int8")
        if not (len(shape) == 4 and v.shape == shape and v.get_device() == d and k.stride()[3] == v.stride()[3] == 1):
            raise ValueError("KVPages: k and v must be [pages, kv_heads, page_size, 128] with contiguous rows, on one device")
        self.kv_dtype = _PAGE_DTYPES[dtype]
        if dtype is torch.bfloat16:
            if k_scale is not None or v_scale is not None:
                raise ValueError("KVPages: bf16 pages take no scales")
        else:
            for s in (k_scale, v_scale):
                if not (s is not None and s.dtype is torch.float32 and s.shape == shape[:3] and s.get_device() == d
                        and (s.stride()[2] == 1 or shape[2] == 1)):
                    raise ValueError("KVPages: 8-bit pages need f32 scales [pages, kv_heads, page_size], contiguous in a page")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def empty(cls, pages: int, kv_heads: int, page_size: int, dtype: torch.dtype = torch.bfloat16,
              device="cuda") -> "KVPages":
        """A zeroed pool of pages."""
        k, v = (torch.zeros((pages, kv_heads, page_size, 128), dtype=dtype, device=device) for _ in range(2))
        if dtype == torch.bfloat16:
            return cls(k, v)
        return cls(k, v, *(torch.zeros((pages, kv_heads, page_size), device=device) for _ in range(2)))

    def _desc(self) -> bytes:
        k, v, ks, vs = self.k, self.v, self.k_scale, self.v_scale
        P, G, ps, D = k.shape
        (k0, k1, k2, _), (v0, v1, v2, _) = k.stride(), v.stride()
        if P == 1:  # torch leaves the stride of a dim of one element open
            k0 = v0 = 16
        if G == 1:
            k1 = v1 = 16
        if ps == 1:
            k2 = v2 = 16
        if ks is None:
            return _PACK_PAGES(k.data_ptr(), v.data_ptr(), 0, 0, P, ps, G, D, self.kv_dtype, k0, k1, k2, v0, v1, v2,
                               0, 0, 0, 0)
        return _PACK_PAGES(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), P, ps, G, D, self.kv_dtype,
                           k0, k1, k2, v0, v1, v2, *_st2(ks), *_st2(vs))


# The wrappers below are called once a layer for single tokens: the checks read
# each attribute once and format no message before it is needed.
def _no_grad(what: str, *ts: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        raise ValueError(f"{what}: no gradient is computed; call it under torch.no_grad()")


def _on(d: int, fn, *args) -> int:
    """fn(*args, stream) on device d's current stream, with d the current device."""
    LAUNCHES[0] += 1
    if d == torch._C._cuda_getDevice():  # (a CUDA tensor is there: CUDA has been initialised)
        return fn(*args, torch._C._cuda_getCurrentRawStream(d))
    with torch.cuda.device(d):
        return fn(*args, torch._C._cuda_getCurrentRawStream(d))


def _batch_desc(what: str, table: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor, rows: int, d: int) -> bytes:
    i32, size, B = torch.int32, table.shape, lens.shape[0] if lens.dim() == 1 else -1
    if not (table.dtype is i32 and cu.dtype is i32 and lens.dtype is i32 and len(size) == 2 and size[0] == B
            and size[1] >= 1 and cu.shape == (B + 1,) and lens.is_contiguous() and cu.is_contiguous()
            and (table.stride()[1] == 1 or size[1] == 1)):
        raise ValueError(f"{what}: page_table [B, max_pages], cu_new [B + 1] and seq_lens [B] must be int32 with contiguous rows")
    if not (table.get_device() == cu.get_device() == lens.get_device() == d):
        raise ValueError(f"{what}: all tensors must be on one device")
    return _PACK_BATCH(table.data_ptr(), table.stride()[0], cu.data_ptr(), lens.data_ptr(), B, size[1], rows)


def _packed(what: str, t: torch.Tensor, heads: int, d: int) -> tuple:
    """Rows of the packed bf16 [rows, heads, 128] on device d, and their strides."""
    size, st = t.shape, t.stride()
    if not (len(size) == 3 and size[1] == heads and size[2] == 128 and t.dtype is torch.bfloat16 and st[2] == 1):
        raise ValueError(f"{what}: packed rows must be bf16 [rows, {heads}, 128] with a contiguous last dim")
    if t.get_device() != d:
        raise ValueError(f"{what}: all tensors must be on one device")
    return size[0], _PACK2(st[0] if size[0] != 1 else 16, st[1] if heads != 1 else 16)


def paged_kv_write(pages: KVPages, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, cu_new: torch.Tensor,
                   seq_lens: torch.Tensor) -> None:
    """Write the packed new rows k, v bf16 [rows, kv_heads, 128] of a batch into
    their pages, quantised with a scale per token and head where the pages are
    8-bit.  Rows [cu_new[b], cu_new[b + 1]) are the last of sequence b's
    seq_lens[b] positions, and position p lies in page page_table[b, p //
    page_size].  All three are int32 on the device, so one captured call serves
    every step.  A slot that two rows land in keeps the later row."""
    G, d = pages.k.shape[1], pages.k.get_device()
    rows, k_st = _packed("paged_kv_write", k, G, d)
    v_rows, v_st = _packed("paged_kv_write", v, G, d)
    if rows != v_rows:
        raise ValueError("paged_kv_write: k and v must have the same number of rows")
    _no_grad("paged_kv_write", k, v)
    batch = _batch_desc("paged_kv_write", page_table, cu_new, seq_lens, rows, d)
    _need_cuda(k)
    L.check(_on(d, L.lib().wf_paged_kv_write, pages._desc(), batch, k.data_ptr(), v.data_ptr(), k_st, v_st),
            "wf_paged_kv_write")


def paged_kv_read(pages: KVPages, page_table: torch.Tensor, cu_new: torch.Tensor, seq_lens: torch.Tensor,
                  rows: int | None = None, out_k: torch.Tensor | None = None, out_v: torch.Tensor | None = None):
    """The inverse of paged_kv_write: positions seq_lens[b] - n_b .. of each
    sequence, n_b = cu_new[b + 1] - cu_new[b], as packed bf16 rows [rows,
    kv_heads, 128] (whole sequences when cu_new is the prefix sum of seq_lens).
    ``rows`` (or the outputs' size) is the packed total; rows behind cu_new[-1]
    are not written."""
    G, d = pages.k.shape[1], pages.k.get_device()
    _check((out_k is None) == (out_v is None), "paged_kv_read: give both outputs or neither")
    if out_k is None:
        _check(rows is not None and rows >= 0, "paged_kv_read: rows is needed without outputs")
        out_k = torch.empty((rows, G, 128), dtype=torch.bfloat16, device=pages.k.device)
        out_v = torch.empty_like(out_k)
        k_st = v_st = _PACK2(G * 128, 128)
    else:
        k_rows, k_st = _packed("paged_kv_read", out_k, G, d)
        v_rows, v_st = _packed("paged_kv_read", out_v, G, d)
        _check(k_rows == v_rows and (rows is None or rows == k_rows), "paged_kv_read: outputs must both hold `rows` rows")
        rows = k_rows
    batch = _batch_desc("paged_kv_read", page_table, cu_new, seq_lens, rows, d)
    _need_cuda(out_k)
    L.check(_on(d, L.lib().wf_paged_kv_read, pages._desc(), batch, out_k.data_ptr(), out_v.data_ptr(), k_st, v_st),
            "wf_paged_kv_read")
    return out_k, out_v


def paged_attention(q: torch.Tensor, pages: KVPages, page_table: torch.Tensor, cu_new: torch.Tensor,
                    seq_lens: torch.Tensor, *, max_new: int | None = None, max_len: int | None = None, block: int = 0,
                    window: int = 0, sink: int = 0, softmax_scale: float | None = None,
                    out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of packed new rows q bf16 [rows, H, 128] over their sequences'
    pages (already holding the rows' own K/V, paged_kv_write); the batch is
    described as there.  H is a multiple of the pages' K/V heads.

    A row at position p sees keys below hi = min(len, (p // block + 1) * block)
    (block 0: the whole sequence; 1: causal; a chunk's tokens: block-causal);
    with window > 0 only the last ``window`` of those and the first ``sink``.
    Rows that see nothing are zero, and what keys that a row does not see hold does
    not matter to it, NaN included (e4m3 NaN codes, which the write never makes, do).
    ``max_new`` / ``max_len`` bound a
    sequence's new rows and length where the caller knows them; they steer the
    split of the work only.  Rows behind cu_new[-1] are not written.  With
    ``return_lse`` also the f32 log-sum-exp [rows, H]."""
    _check(q.dim() == 3, "paged_attention: q must be packed rows [rows, H, 128]")
    H, d = q.shape[1], q.get_device()
    rows, q_st = _packed("paged_attention", q, H, d)
    _no_grad("paged_attention", q)
    _, G, ps, _ = pages.k.shape
    if pages.k.get_device() != d:
        raise ValueError("paged_attention: all tensors must be on one device")
    _check(H % G == 0, "paged_attention: query heads must be a multiple of the K/V heads")
    if not (0 <= block <= _I32 and 0 <= window <= _I32 and 0 <= sink <= _I32):  # ctypes would cut them off
        raise ValueError("paged_attention: block, window and sink must be 0 to 2^31 - 1")
    batch = _batch_desc("paged_attention", page_table, cu_new, seq_lens, rows, d)
    if out is None:
        out = q.new_empty((rows, H, 128))
        o_st = _PACK2(H * 128, 128)
    else:
        o_rows, o_st = _packed("paged_attention", out, H, d)
        _check(o_rows == rows, "paged_attention: out must match q")
    _need_cuda(q)
    lse = q.new_empty((rows, H), dtype=torch.float32) if return_lse else None
    max_new = rows if max_new is None else int(max_new)
    max_len = page_table.shape[1] * ps if max_len is None else int(max_len)
    desc = pages._desc()
    lib = L.lib()
    need = lib.wf_paged_attn_workspace(desc, batch, H, window, sink, max_new, max_len)
    ws = q.new_empty((need,), dtype=torch.uint8) if need > 0 else None
    scale = _SCALE if softmax_scale is None else float(softmax_scale)
    L.check(_on(d, lib.wf_paged_attn, desc, batch, q.data_ptr(), q_st, out.data_ptr(), o_st,
                lse.data_ptr() if lse is not None else None, H, block, window, sink, max_new, max_len, scale,
                ws.data_ptr() if ws is not None else None, need), "wf_paged_attn")
    return (out, lse) if return_lse else out


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lens: torch.Tensor | None = None,
                    key_mask: torch.Tensor | None = None, kv_index: torch.Tensor | None = None,
                    softmax_scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of q bf16 [B, Lq, H, 128] to an encoder's states k, v [N, Lk,
    kv_heads, 128] of another length.  Entry b attends to states kv_index[b]
    (int32 [B]; without it N is B, or 1 for states that all share), there to
    the keys below kv_lens[n] (int32 [N]) that key_mask [N, Lk] (bool) keeps;
    what the other keys hold does not matter.  Queries left without keys give
    zeros.  With ``return_lse`` also the f32 log-sum-exp [B, Lq, H]."""
    size, bf = k.shape, torch.bfloat16
    if not (q.dim() == 4 and len(size) == 4 and v.shape == size and q.dtype is bf and k.dtype is bf and v.dtype is bf
            and q.shape[3] == size[3] and q.stride()[3] == k.stride()[3] == v.stride()[3] == 1):
        raise ValueError("cross_attention: q [B, Lq, H, 128] and k, v [N, Lk, kv_heads, 128] must be bf16 with contiguous "
                         "last dims")
    B, Lq, H, D = q.shape
    N, Lk, G, _ = size
    d = q.get_device()
    _check(N >= 1 and Lk >= 1 and G >= 1 and H % G == 0,
           "cross_attention: query heads must be a multiple of the K/V heads, states not empty")
    _check(kv_index is not None or N == 1 or N == B, "cross_attention: N states for B entries need kv_index")
    for t, n in ((kv_index, B), (kv_lens, N)):
        _check(t is None or (t.dtype is torch.int32 and t.shape == (n,) and t.is_contiguous() and t.get_device() == d),
               "cross_attention: kv_index [B] and kv_lens [N] must be contiguous int32 on q's device")
    _check(key_mask is None or (key_mask.dtype is torch.bool and key_mask.shape == (N, Lk) and key_mask.get_device() == d
                                and (key_mask.stride()[1] == 1 or Lk == 1)),
           "cross_attention: key_mask must be bool [N, Lk] with contiguous rows on q's device")
    _no_grad("cross_attention", q, k, v)
    if out is None:
        out = q.new_empty((B, Lq, H, D))
    if not (out.shape == q.shape and out.dtype is bf and out.stride()[3] == 1
            and out.get_device() == k.get_device() == v.get_device() == d):
        raise ValueError("cross_attention: out must match q, all tensors on one device")
    _need_cuda(q)
    lse = q.new_empty((B, Lq, H), dtype=torch.float32) if return_lse else None
    lib = L.lib()
    need = lib.wf_cross_attn_workspace(B, Lq, N, Lk, H, G)
    ws = q.new_empty((need,), dtype=torch.uint8) if need > 0 else None
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    L.check(_on(d, lib.wf_cross_attn, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                lse.data_ptr() if lse is not None else None, B, Lq, N, Lk, H, G, D, _PACK3(*_st3(q)),
                _PACK3(*_st3(k)), _PACK3(*_st3(v)), _PACK3(*_st3(out)),
                kv_index.data_ptr() if kv_index is not None else None,
                kv_lens.data_ptr() if kv_lens is not None else None,
                key_mask.data_ptr() if key_mask is not None else None,
                key_mask.stride(0) if key_mask is not None else 0, scale,
                ws.data_ptr() if ws is not None else None, need), "wf_cross_attn")
    return (out, lse) if return_lse else out
