"""PyTorch-facing op surface: same names, argument order, dtypes, shapes and return conventions
as the reference extension ``int4_native_tc_ops`` (``int4_native_tc/csrc/bindings.cpp:208-309``).

PyTorch is only plumbing here: it owns the device memory and the stream; every op is one or more
calls into the C-ABI library.  Quantise ops allocate and return their outputs, scaled GEMMs write
into the caller's ``out`` and return ``None`` -- the reference's ownership rules
(``int4_quant.cu:209-212``, ``int4_gemm.cu:831-837``).
"""
from __future__ import annotations

import math
import struct

import torch

from . import _cabi
from ._cabi import check, lib

_DTYPES = {torch.bfloat16: _cabi.BF16, torch.float16: _cabi.FP16, torch.float32: _cabi.FP32}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _dev(t: torch.Tensor) -> int:
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def _stream(t: torch.Tensor) -> int:
    """Handle of torch's current stream on the tensor's device (the stream the reference launches on)."""
    if _raw_stream is not None:
        return _raw_stream(_dev(t))
    return torch.cuda.current_stream(t.device).cuda_stream


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _cuda2d(t: torch.Tensor, name: str) -> None:
    _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be CUDA tensor")
    _require(t.dim() == 2, f"{name} must be 2D")


def _float_input(t: torch.Tensor, name: str) -> torch.Tensor:
    _require(t.dtype in _DTYPES, f"{name} must be bfloat16, float16 or float32")
    if t.stride(1) != 1 or (t.stride(0) * t.element_size()) % 16 != 0 or t.data_ptr() % 16 != 0:
        t = t.contiguous()
    return t


def _same_device(*ts: torch.Tensor) -> None:
    d = ts[0].device
    for t in ts[1:]:
        _require(t.device == d, "all tensors must be on the same device")


def _packed(t: torch.Tensor, name: str) -> torch.Tensor:
    _require(t.is_cuda, f"{name} must be CUDA tensor")
    _require(t.dtype == torch.uint8, f"{name} must be uint8")
    _require(t.is_contiguous(), f"{name} must be contiguous")
    return t


def _f32(t: torch.Tensor, name: str, numel: int) -> torch.Tensor:
    _require(t.is_cuda and t.dtype == torch.float32, f"{name} must be a float32 CUDA tensor")
    _require(t.is_contiguous(), f"{name} must be contiguous")
    _require(t.numel() == numel, f"{name} has {t.numel()} elements, expected {numel}")
    return t


# --------------------------------------------------------------------------- #
# quantise / pack
# --------------------------------------------------------------------------- #
def _quant_rowwise(x: torch.Tensor, role: int, who: str):
    _cuda2d(x, "input" if role == _cabi.ROLE_ACTIVATION else "weight")
    R, K = x.shape
    _require(K % 2 == 0, "K must be even for INT4 packing")
    x = _float_input(x, who)
    packed = torch.empty((R, K // 2), dtype=torch.uint8, device=x.device)
    scale = torch.empty((R,), dtype=torch.float32, device=x.device)
    check(lib.i4tc_quant_rowwise(x.data_ptr(), _DTYPES[x.dtype], R, K, x.stride(0), packed.data_ptr(),
                                 scale.data_ptr(), role, _dev(x), _stream(x)), who)
    return packed, scale


def _quant_grouped(x: torch.Tensor, group_size: int, role: int, who: str):
    _cuda2d(x, "input" if role == _cabi.ROLE_ACTIVATION else "weight")
    R, K = x.shape
    group_size = int(group_size)
    _require(group_size > 0 and K % group_size == 0, "K must be divisible by group_size")
    _require(group_size % 2 == 0, "group_size must be even")
    x = _float_input(x, who)
    G = K // group_size
    packed = torch.empty((G, R, group_size // 2), dtype=torch.uint8, device=x.device)
    scale = torch.empty((G, R), dtype=torch.float32, device=x.device)
    check(lib.i4tc_quant_grouped(x.data_ptr(), _DTYPES[x.dtype], R, K, x.stride(0), group_size,
                                 packed.data_ptr(), scale.data_ptr(), role, _dev(x), _stream(x)), who)
    return packed, scale


def dynamic_int4_quant(input: torch.Tensor):
    """[M,K] -> (packed u8 [M,K/2], scale f32 [M]).  Reference: ``int4_quant.cu:201``."""
    return _quant_rowwise(input, _cabi.ROLE_ACTIVATION, "dynamic_int4_quant")


def static_int4_weight_quant(weight: torch.Tensor):
    """[N,K] -> (packed u8 [N,K/2], scale f32 [N]).  Reference: ``int4_quant.cu:289``."""
    return _quant_rowwise(weight, _cabi.ROLE_WEIGHT, "static_int4_weight_quant")


def dynamic_int4_quant_grouped(input: torch.Tensor, group_size: int):
    """[M,K] -> (packed u8 [G,M,gs/2], scale f32 [G,M]).  Reference: ``int4_quant.cu:806``."""
    return _quant_grouped(input, group_size, _cabi.ROLE_ACTIVATION, "dynamic_int4_quant_grouped")


def static_int4_weight_quant_grouped(weight: torch.Tensor, group_size: int):
    """[N,K] -> (packed u8 [G,N,gs/2], scale f32 [G,N]).  Reference: ``int4_quant.cu:712``."""
    return _quant_grouped(weight, group_size, _cabi.ROLE_WEIGHT, "static_int4_weight_quant_grouped")


def _ext_input(input: torch.Tensor, group_size: int, who: str):
    _cuda2d(input, "input")
    _require(input.dtype in (torch.bfloat16, torch.float16), f"{who}: input must be bfloat16 or float16")
    M, K = input.shape
    _require(group_size > 0 and K % group_size == 0, "K must be divisible by group_size")
    _require(group_size % 2 == 0, "group_size must be even")
    if input.stride(1) != 1:
        input = input.contiguous()
    return input, M, K, K // group_size


def dynamic_int4_quant_clipped_grouped(input: torch.Tensor, group_size: int, clip_ratio: float):
    """[M,K] -> (packed u8 [G,M,gs/2], scale f32 [G,M]) with the range ``absmax * clip_ratio`` per group.
    Reference: ``int4_quant.cu:906`` (checks ``:909-916``)."""
    x, M, K, G = _ext_input(input, group_size, "dynamic_int4_quant_clipped_grouped")
    _require(0.0 < clip_ratio <= 1.0, "clip_ratio must be in (0, 1]")
    packed = torch.empty((G, M, group_size // 2), dtype=torch.uint8, device=x.device)
    scale = torch.empty((G, M), dtype=torch.float32, device=x.device)
    check(lib.i4tc_quant_clipped_grouped(x.data_ptr(), _DTYPES[x.dtype], M, K, x.stride(0), int(group_size),
                                         float(clip_ratio), packed.data_ptr(), scale.data_ptr(), _dev(x),
                                         _stream(x)), "dynamic_int4_quant_clipped_grouped")
    return packed, scale


def dynamic_int4_quant_asymmetric_clipped_grouped(input: torch.Tensor, group_size: int, clip_ratio: float,
                                                  smooth_scale: torch.Tensor | None = None):
    """[M,K] -> (packed u8 [G,M,gs/2], scale f32 [G,M], azp_adj f32 [G,M]); asymmetric codes stored as
    ``u - 8``, optional division by ``smooth_scale`` [K] (same dtype as the input) and symmetric clipping first.
    Reference: ``int4_quant.cu:1433`` (checks ``:1437-1470``)."""
    who = "dynamic_int4_quant_asymmetric_clipped_grouped"
    x, M, K, G = _ext_input(input, group_size, who)
    _require(0.0 < clip_ratio <= 1.0, "clip_ratio must be in (0, 1]")
    sm_ptr = None
    if smooth_scale is not None:
        _require(smooth_scale.is_cuda and smooth_scale.dtype == x.dtype, "smooth_scale must match the input's dtype")
        _require(smooth_scale.numel() == K, "smooth_scale must be [K]")
        _same_device(x, smooth_scale)
        smooth_scale = smooth_scale.contiguous()
        sm_ptr = smooth_scale.data_ptr()
    packed = torch.empty((G, M, group_size // 2), dtype=torch.uint8, device=x.device)
    scale = torch.empty((G, M), dtype=torch.float32, device=x.device)
    azp_adj = torch.empty((G, M), dtype=torch.float32, device=x.device)
    check(lib.i4tc_quant_asymmetric_grouped(x.data_ptr(), _DTYPES[x.dtype], M, K, x.stride(0), int(group_size),
                                            float(clip_ratio), sm_ptr, packed.data_ptr(), scale.data_ptr(),
                                            azp_adj.data_ptr(), _dev(x), _stream(x)), who)
    return packed, scale, azp_adj


def dynamic_int4_quant_asymmetric_grouped(input: torch.Tensor, group_size: int):
    """[M,K] -> (packed, scale, azp_adj) without clipping or smoothing.  Reference: ``int4_quant.cu:1262``."""
    return dynamic_int4_quant_asymmetric_clipped_grouped(input, group_size, 1.0, None)


def int4_weight_group_sums(b_packed: torch.Tensor) -> torch.Tensor:
    """Group-major packed weights u8 [G,N,gs/2] -> ``w_col_sum`` f32 [G,N], the sum of each group's codes (the
    operand the reference's callers build in torch, ``int4_native_tc/profile_layer.py:96-119``)."""
    _packed(b_packed, "b_packed")
    _require(b_packed.dim() == 3 and b_packed.shape[2] % 4 == 0, "b_packed must be [G, N, gs/2] with gs % 8 == 0")
    G, N, half = b_packed.shape
    out = torch.empty((G, N), dtype=torch.float32, device=b_packed.device)
    check(lib.i4tc_weight_group_sums(b_packed.data_ptr(), G * N, 2 * half, out.data_ptr(), _dev(out),
                                     _stream(out)), "int4_weight_group_sums")
    return out


def rmsnorm_int4_quant_grouped(input: torch.Tensor, norm_weight: torch.Tensor, eps: float, group_size: int = 128):
    """RMSNorm fused in front of the grouped quantiser (no reference op; the reference's report names the fusion as
    its follow-up).  bf16 [M,K], bf16 [K] -> (packed u8 [G,M,gs/2], scale f32 [G,M]) of
    ``bf16(bf16(x * rsqrt(mean(x^2) + eps)) * norm_weight)``."""
    _cuda2d(input, "input")
    _require(input.dtype == torch.bfloat16 and norm_weight.dtype == torch.bfloat16, "input and norm_weight must be bfloat16")
    _require(input.stride(1) == 1, "input rows must be contiguous")
    _same_device(input, norm_weight)
    M, K = input.shape
    _require(norm_weight.is_contiguous() and norm_weight.numel() == K, "norm_weight must be a contiguous [K] tensor")
    _require(group_size > 0 and K % group_size == 0, "K must be divisible by group_size")
    G = K // group_size
    packed = torch.empty((G, M, group_size // 2), dtype=torch.uint8, device=input.device)
    scale = torch.empty((G, M), dtype=torch.float32, device=input.device)
    check(lib.i4tc_rmsnorm_quant_grouped(input.data_ptr(), M, K, input.stride(0), norm_weight.data_ptr(), float(eps),
                                         int(group_size), packed.data_ptr(), scale.data_ptr(), _dev(input),
                                         _stream(input)), "rmsnorm_int4_quant_grouped")
    return packed, scale


def rmsnorm(input: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """``bf16(bf16(x * rsqrt(mean(x^2) + eps)) * weight)`` over the last dimension of contiguous bf16 rows."""
    _require(input.is_cuda and input.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16, "input and weight must be bfloat16 CUDA tensors")
    _require(input.is_contiguous() and weight.is_contiguous() and weight.numel() == input.shape[-1], "input and weight must be contiguous")
    _same_device(input, weight)
    out = torch.empty_like(input)
    K = input.shape[-1]
    check(lib.i4tc_rmsnorm(input.data_ptr(), input.numel() // K if K else 0, K, K, weight.data_ptr(), float(eps), out.data_ptr(),
                           _dev(input), _stream(input)), "rmsnorm")
    return out


def qk_norm_rope_(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                  q_heads: int, kv_heads: int, seq: int, eps: float) -> torch.Tensor:
    """In place on the query and key heads (of 128) of contiguous bf16 ``qkv`` [tokens, heads * 128]: RMSNorm per head, then
    the rotary embedding at position ``token % seq`` (tables bf16 [seq, 64])."""
    _cuda2d(qkv, "qkv")
    for t in (qkv, q_weight, k_weight, cos, sin):
        _require(t.dtype == torch.bfloat16 and t.is_contiguous(), "operands must be contiguous bfloat16")
    _same_device(qkv, q_weight, k_weight, cos, sin)
    _require(q_weight.numel() == 128 and k_weight.numel() == 128, "heads must have 128 elements")
    _require(cos.numel() == seq * 64 and sin.numel() == seq * 64, "cos and sin must be [seq, 64]")
    check(lib.i4tc_qk_norm_rope(qkv.data_ptr(), qkv.shape[0], qkv.shape[1], q_heads, kv_heads, seq, q_weight.data_ptr(),
                                k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(), float(eps), _dev(qkv), _stream(qkv)),
          "qk_norm_rope_")
    return qkv


def int4_quant_with_scales(input: torch.Tensor, scale: torch.Tensor, group_size: int = 0):
    """Quantise with caller-supplied divisors (no reference op; the "identical scales" form used to
    compare codes bit for bit).  ``scale`` [M] -> packed [M,K/2]; ``scale`` [G,M] -> packed [G,M,gs/2]."""
    _cuda2d(input, "input")
    R, K = input.shape
    x = _float_input(input, "int4_quant_with_scales")
    _same_device(x, scale)
    if group_size:
        G = K // group_size
        _f32(scale, "scale", G * R)
        packed = torch.empty((G, R, group_size // 2), dtype=torch.uint8, device=x.device)
    else:
        _f32(scale, "scale", R)
        packed = torch.empty((R, K // 2), dtype=torch.uint8, device=x.device)
    check(lib.i4tc_quant_with_scales(x.data_ptr(), _DTYPES[x.dtype], R, K, x.stride(0), int(group_size),
                                     scale.data_ptr(), packed.data_ptr(), _dev(x), _stream(x)),
          "int4_quant_with_scales")
    return packed


def unpack_int4_to_int8(packed: torch.Tensor, K: int) -> torch.Tensor:
    """packed u8 [N,K/2] -> int8 [N,K].  Reference: ``int4_quant.cu:593``."""
    _require(packed.is_cuda, "packed must be CUDA tensor")
    _require(packed.dim() == 2, "packed must be 2D [N, K/2]")
    _require(packed.dtype == torch.uint8, "packed must be uint8")
    _require(packed.size(1) * 2 == K, "packed.size(1) must equal K/2")
    packed = packed.contiguous()
    N = packed.size(0)
    out = torch.empty((N, K), dtype=torch.int8, device=packed.device)
    check(lib.i4tc_unpack_int4_to_int8(packed.data_ptr(), N, K, out.data_ptr(), _dev(packed), _stream(packed)),
          "unpack_int4_to_int8")
    return out


# --------------------------------------------------------------------------- #
# GEMMs
# --------------------------------------------------------------------------- #
def cutlass_int4_gemm(a_packed: torch.Tensor, b_packed: torch.Tensor, M: int, N: int, K: int) -> torch.Tensor:
    """int32 [M,N] = A[M,K] . B[N,K]^T over packed int4.  Reference: ``int4_gemm.cu:779``."""
    _packed(a_packed, "a_packed")
    _packed(b_packed, "b_packed")
    _same_device(a_packed, b_packed)
    _require(K % 64 == 0, "K must be a multiple of 64")
    _require(a_packed.numel() == M * (K // 2), "a_packed does not have M*K/2 bytes")
    _require(b_packed.numel() == N * (K // 2), "b_packed does not have N*K/2 bytes")
    out = torch.empty((M, N), dtype=torch.int32, device=a_packed.device)
    check(lib.i4tc_gemm_int32(a_packed.data_ptr(), b_packed.data_ptr(), out.data_ptr(), M, N, K,
                              _dev(a_packed), _stream(a_packed)), "cutlass_int4_gemm")
    return out


def cutlass_int4_scaled_mm(a_packed, b_packed, scale_a, scale_b, out, M: int, N: int, K: int) -> None:
    """out[m,n] = cast((acc * scale_b[n]) * scale_a[m]) into the caller's bf16/fp16 ``out``.
    Reference: ``int4_gemm.cu:831``."""
    _packed(a_packed, "a_packed")
    _packed(b_packed, "b_packed")
    _same_device(a_packed, b_packed, scale_a, scale_b, out)
    _require(K % 64 == 0, "K must be a multiple of 64")
    _require(out.dtype in (torch.bfloat16, torch.float16), "out must be bfloat16 or float16")
    _require(out.is_contiguous() and out.numel() == M * N, "out must be a contiguous [M,N] tensor")
    _require(a_packed.numel() == M * (K // 2), "a_packed does not have M*K/2 bytes")
    _require(b_packed.numel() == N * (K // 2), "b_packed does not have N*K/2 bytes")
    _f32(scale_a, "scale_a", M)
    _f32(scale_b, "scale_b", N)
    check(lib.i4tc_gemm_scaled(a_packed.data_ptr(), b_packed.data_ptr(), scale_a.data_ptr(), scale_b.data_ptr(),
                               out.data_ptr(), _DTYPES[out.dtype], M, N, K, _dev(out), _stream(out)),
          "cutlass_int4_scaled_mm")


def dynamic_int8_quant(input: torch.Tensor):
    """[M,K] float -> (int8 [M,K], fp32 scale [M]): per-token symmetric int8, ``scale = max(absmax / 127, 1/(127*512))``.
    Reference: ``int4_quant.cu:511`` (kernel ``:432``)."""
    _cuda2d(input, "input")
    x = _float_input(input, "input")
    M, K = x.shape
    q = torch.empty((M, K), dtype=torch.int8, device=x.device)
    scale = torch.empty((M,), dtype=torch.float32, device=x.device)
    check(lib.i4tc_quant_rowwise_int8(x.data_ptr(), _DTYPES[x.dtype], M, K, x.stride(0), q.data_ptr(), scale.data_ptr(),
                                      _dev(x), _stream(x)), "dynamic_int8_quant")
    return q, scale


def cutlass_w4a8_scaled_mm(a, b_int8, scale_a, scale_b, out, M: int, N: int, K: int) -> None:
    """``out[m,n] = cast((sum_k a[m,k] * b_int8[n,k]) * scale_b[n] * scale_a[m])`` with int8 ``a`` [M,K] and the int4
    weight held as int8 ``b_int8`` [N,K] (``unpack_int4_to_int8``).  Reference: ``int4_gemm.cu:874-899``."""
    _require(a.is_cuda and b_int8.is_cuda, "Inputs must be CUDA")
    _require(scale_a.is_cuda and scale_b.is_cuda, "Scales must be CUDA")
    _require(out.is_cuda, "Output must be CUDA")
    _require(K % 32 == 0, "K must be multiple of 32 for INT8 alignment")
    _require(a.dtype == torch.int8, "a must be int8")
    _require(b_int8.dtype == torch.int8, "b_int8 must be int8")
    _require(out.dtype in (torch.bfloat16, torch.float16),
             "cutlass_w4a8_scaled_mm: unsupported output dtype, must be bfloat16 or float16")
    _same_device(a, b_int8, scale_a, scale_b, out)
    _require(a.is_contiguous() and a.numel() == M * K, "a must be a contiguous [M,K] tensor")
    _require(b_int8.is_contiguous() and b_int8.numel() == N * K, "b_int8 must be a contiguous [N,K] tensor")
    _require(out.is_contiguous() and out.numel() == M * N, "out must be a contiguous [M,N] tensor")
    _f32(scale_a, "scale_a", M)
    _f32(scale_b, "scale_b", N)
    check(lib.i4tc_gemm_w4a8_scaled(a.data_ptr(), b_int8.data_ptr(), scale_a.data_ptr(), scale_b.data_ptr(),
                                    out.data_ptr(), _DTYPES[out.dtype], M, N, K, _dev(out), _stream(out)),
          "cutlass_w4a8_scaled_mm")


def _grouped_gemm(a_packed, b_packed, scale_a, scale_b, azp_adj, w_col_sum, out, M, N, group_size, num_groups, who) -> None:
    """The per-group GEMM, with scratch from torch's caching allocator where the library asks for some (large M).  When
    there is no memory for it the library's kernel without scratch serves the call."""
    dev = _dev(out)
    scratch, nbytes = None, 0
    if M > 128:
        nbytes = lib.i4tc_gemm_grouped_scratch_bytes(M, N, num_groups, azp_adj is not None, dev)
        if nbytes:
            try:
                scratch = torch.empty(nbytes, dtype=torch.uint8, device=out.device)
            except torch.cuda.OutOfMemoryError:
                nbytes = 0
    check(lib.i4tc_gemm_grouped_scratch(a_packed.data_ptr(), b_packed.data_ptr(), scale_a.data_ptr(), scale_b.data_ptr(),
                                        None if azp_adj is None else azp_adj.data_ptr(),
                                        None if w_col_sum is None else w_col_sum.data_ptr(), out.data_ptr(), M, N,
                                        group_size, num_groups, None if scratch is None else scratch.data_ptr(), nbytes,
                                        dev, _stream(out)), who)


def _pad256(n: int) -> int:
    return (n + 255) & ~255


def linear(x: torch.Tensor, w_packed: torch.Tensor, w_scale: torch.Tensor, N: int, per_channel: bool) -> torch.Tensor:
    """Quantise the activations [M,K] and multiply, as ``dynamic_int4_quant(_grouped)`` + ``cutlass_int4_scaled_mm`` /
    ``cutlass_int4_fused_grouped_gemm`` do, through one library call and one buffer for codes, scales and scratch (a single
    token spends 20 us of host time in the separate ops).  bf16 [M,N]."""
    _cuda2d(x, "input")
    M, K = x.shape
    if per_channel:
        _require(K % 64 == 0, "K must be a multiple of 64")
    else:
        _require(K % 128 == 0, "K must be divisible by group_size")
    x = _float_input(x, "input")
    groups = 1 if per_channel else K // 128
    _packed(w_packed, "b_packed")
    _require(w_packed.numel() == N * (K // 2), "b_packed does not have N*K/2 bytes")
    _f32(w_scale, "scale_b", groups * N)
    dev = _dev(x)
    _require(w_packed.device == x.device and w_scale.device == x.device, "all tensors must be on the same device")
    out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    packed_bytes = _pad256(M * (K // 2))
    base_bytes = packed_bytes + _pad256(groups * M * 4)
    extra = lib.i4tc_gemm_grouped_scratch_bytes(M, N, groups, 0, dev) if M > 128 and not per_channel else 0
    if extra:
        try:
            buf = torch.empty(base_bytes + extra, dtype=torch.uint8, device=x.device)
        except torch.cuda.OutOfMemoryError:
            extra = 0
    if not extra:
        buf = torch.empty(base_bytes, dtype=torch.uint8, device=x.device)
    at = buf.data_ptr()
    check(lib.i4tc_linear(x.data_ptr(), _DTYPES[x.dtype], M, K, x.stride(0), w_packed.data_ptr(), w_scale.data_ptr(),
                          int(per_channel), at, at + packed_bytes, out.data_ptr(), N, at + base_bytes if extra else None,
                          extra, dev, _stream(x)), "linear")
    return out


def linear_asymmetric(x: torch.Tensor, w_packed: torch.Tensor, w_scale: torch.Tensor, w_col_sum: torch.Tensor, N: int,
                      clip_ratio: float, smooth_scale: torch.Tensor | None = None) -> torch.Tensor:
    """``dynamic_int4_quant_asymmetric_clipped_grouped`` + ``cutlass_int4_fused_grouped_gemm_azp`` in one library call and one
    buffer, as ``linear`` does for symmetric codes.  bf16 [M,N]."""
    x, M, K, G = _ext_input(x, 128, "dynamic_int4_quant_asymmetric_clipped_grouped")
    _require(0.0 < clip_ratio <= 1.0, "clip_ratio must be in (0, 1]")
    sm_ptr = None
    if smooth_scale is not None:
        _require(smooth_scale.is_cuda and smooth_scale.dtype == x.dtype, "smooth_scale must match the input's dtype")
        _require(smooth_scale.numel() == K, "smooth_scale must be [K]")
        _same_device(x, smooth_scale)
        smooth_scale = smooth_scale.contiguous()
        sm_ptr = smooth_scale.data_ptr()
    _packed(w_packed, "b_packed")
    _require(w_packed.numel() == N * (K // 2), "b_packed must be [G, N, 64]")
    _f32(w_scale, "scale_b", G * N)
    _f32(w_col_sum, "w_col_sum", G * N)
    _same_device(x, w_packed, w_scale, w_col_sum)
    dev = _dev(x)
    out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    codes, values = _pad256(M * (K // 2)), _pad256(G * M * 4)
    base_bytes = codes + 2 * values
    extra = lib.i4tc_gemm_grouped_scratch_bytes(M, N, G, 1, dev) if M > 128 else 0
    if extra:
        try:
            buf = torch.empty(base_bytes + extra, dtype=torch.uint8, device=x.device)
        except torch.cuda.OutOfMemoryError:
            extra = 0
    if not extra:
        buf = torch.empty(base_bytes, dtype=torch.uint8, device=x.device)
    at = buf.data_ptr()
    check(lib.i4tc_linear_asymmetric(x.data_ptr(), _DTYPES[x.dtype], M, K, x.stride(0), float(clip_ratio), sm_ptr, w_packed.data_ptr(),
                                     w_scale.data_ptr(), w_col_sum.data_ptr(), at, at + codes, at + codes + values, out.data_ptr(),
                                     N, at + base_bytes if extra else None, extra, dev, _stream(x)), "linear_asymmetric")
    return out


def cutlass_int4_fused_grouped_gemm(a_packed, b_packed, scale_a, scale_b, out, M: int, N: int,
                                    group_size: int, num_groups: int) -> None:
    """Per-group-128 fused linear into the caller's bf16 ``out`` [M,N].
    Reference: ``int4_gemm.cu:4231`` (checks at ``:4243-4252``)."""
    _packed(a_packed, "a_packed")
    _packed(b_packed, "b_packed")
    _same_device(a_packed, b_packed, scale_a, scale_b, out)
    _require(group_size == 128, "fused grouped GEMM only supports group_size=128")
    _require(out.dtype == torch.bfloat16, "fused grouped GEMM only supports BF16 output")
    _require(out.is_contiguous() and out.numel() == M * N, "out must be a contiguous [M,N] tensor")
    _require(a_packed.numel() == num_groups * M * 64, "a_packed must be [G, M, 64]")
    _require(b_packed.numel() == num_groups * N * 64, "b_packed must be [G, N, 64]")
    _f32(scale_a, "scale_a", num_groups * M)
    _f32(scale_b, "scale_b", num_groups * N)
    _grouped_gemm(a_packed, b_packed, scale_a, scale_b, None, None, out, M, N, group_size, num_groups,
                  "cutlass_int4_fused_grouped_gemm")


# Same contract, different kernels in the reference (int4_gemm.cu:3751, 4073, 4007, 3932).
cutlass_int4_fused_grouped_gemm_v5 = cutlass_int4_fused_grouped_gemm
cutlass_int4_fused_grouped_gemm_v7 = cutlass_int4_fused_grouped_gemm
cutlass_int4_fused_grouped_gemm_v8 = cutlass_int4_fused_grouped_gemm
cutlass_int4_fused_grouped_gemm_v9 = cutlass_int4_fused_grouped_gemm


def cutlass_int4_scaled_mm_grouped(a_packed, b_packed, scale_a, scale_b, out, M: int, N: int, group_size: int,
                                   num_groups: int) -> None:
    """The reference's per-group loop of scaled GEMMs (``int4_gemm.cu:929-992``), served here by the fused kernel:
    a narrower contract -- ``group_size`` 128 and bf16 output only, and no rounding of each group's product to the
    output type before the fp32 accumulation (the reference's loop accepts any multiple of 64 and fp16)."""
    _require(group_size == 128, "cutlass_int4_scaled_mm_grouped: this build serves group_size=128 only "
                                f"(got {group_size}; the reference accepts any multiple of 64)")
    _require(out.dtype == torch.bfloat16, "cutlass_int4_scaled_mm_grouped: this build writes bfloat16 only "
                                         f"(got {out.dtype}; the reference also accepts float16)")
    cutlass_int4_fused_grouped_gemm(a_packed, b_packed, scale_a, scale_b, out, M, N, group_size, num_groups)


def cutlass_int4_fused_grouped_gemm_azp(a_packed, b_packed, scale_a, scale_b, out, azp_adj, w_col_sum, M: int,
                                        N: int, group_size: int, num_groups: int) -> None:
    """Per-group-128 fused linear with the zero-point term of asymmetric activations into the caller's bf16
    ``out`` [M,N]: ``sum_g sa*sb*(acc_g + azp_adj[g,m]*w_col_sum[g,n])``.  Reference: ``int4_gemm.cu:4298``."""
    _packed(a_packed, "a_packed")
    _packed(b_packed, "b_packed")
    _same_device(a_packed, b_packed, scale_a, scale_b, out, azp_adj, w_col_sum)
    _require(group_size == 128, "fused grouped GEMM only supports group_size=128")
    _require(out.dtype == torch.bfloat16, "cutlass_int4_fused_grouped_gemm_azp currently supports BF16 output only")
    _require(out.is_contiguous() and out.numel() == M * N, "out must be a contiguous [M,N] tensor")
    _require(a_packed.numel() == num_groups * M * 64, "a_packed must be [G, M, 64]")
    _require(b_packed.numel() == num_groups * N * 64, "b_packed must be [G, N, 64]")
    _f32(scale_a, "scale_a", num_groups * M)
    _f32(scale_b, "scale_b", num_groups * N)
    _f32(azp_adj, "azp_adj", num_groups * M)
    _f32(w_col_sum, "w_col_sum", num_groups * N)
    _grouped_gemm(a_packed, b_packed, scale_a, scale_b, azp_adj, w_col_sum, out, M, N, group_size, num_groups,
                  "cutlass_int4_fused_grouped_gemm_azp")


# Same contract, different kernels in the reference (int4_gemm.cu:3838, 4149).
cutlass_int4_fused_grouped_gemm_v5_azp = cutlass_int4_fused_grouped_gemm_azp
cutlass_int4_fused_grouped_gemm_v7_azp = cutlass_int4_fused_grouped_gemm_azp


def cutlass_int4_scaled_mm_azp_grouped(a_packed, b_packed, scale_a, scale_b, out, azp_adj, w_col_sum, M: int, N: int,
                                       group_size: int, num_groups: int) -> None:
    """The reference's per-group loop with the zero-point term (``int4_gemm.cu:994-1000``), served by the fused
    kernel under the same narrower contract as ``cutlass_int4_scaled_mm_grouped``."""
    _require(group_size == 128, "cutlass_int4_scaled_mm_azp_grouped: this build serves group_size=128 only "
                                f"(got {group_size}; the reference accepts any multiple of 64)")
    _require(out.dtype == torch.bfloat16, "cutlass_int4_scaled_mm_azp_grouped: this build writes bfloat16 only "
                                         f"(got {out.dtype}; the reference also accepts float16)")
    cutlass_int4_fused_grouped_gemm_azp(a_packed, b_packed, scale_a, scale_b, out, azp_adj, w_col_sum, M, N, group_size,
                                        num_groups)


def int4_grouped_partials(a_packed, b_packed, M: int, N: int, num_groups: int) -> torch.Tensor:
    """int32 [G,M,N]: the per-group integer accumulators of the fused kernel (no reference op)."""
    _packed(a_packed, "a_packed")
    _packed(b_packed, "b_packed")
    _same_device(a_packed, b_packed)
    _require(a_packed.numel() == num_groups * M * 64, "a_packed must be [G, M, 64]")
    _require(b_packed.numel() == num_groups * N * 64, "b_packed must be [G, N, 64]")
    out = torch.empty((num_groups, M, N), dtype=torch.int32, device=a_packed.device)
    check(lib.i4tc_gemm_grouped_int32(a_packed.data_ptr(), b_packed.data_ptr(), out.data_ptr(), M, N,
                                      num_groups, _dev(out), _stream(out)), "int4_grouped_partials")
    return out


# --------------------------------------------------------------------------- #
# decoding: a few tokens over 4-bit weights and a paged cache (no reference ops)
# --------------------------------------------------------------------------- #
def _half_input(t: torch.Tensor, name: str, dim: int) -> None:
    _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be CUDA tensor")
    _require(t.dim() == dim, f"{name} must be {dim}D")
    _require(t.dtype == torch.bfloat16 or t.dtype == torch.float16, f"{name} must be bfloat16 or float16")
    _require(not (t.requires_grad and torch.is_grad_enabled()), f"{name} requires grad: the op has no backward pass, call it under torch.no_grad()")


# Arguments of an entry point that takes a struct: one conversion for all of them.
_W4A16_ARGS = struct.Struct("@4P7q").pack
_ROPE_ARGS = struct.Struct("@4P12qd").pack
_ATTENTION_ARGS = struct.Struct("@10P21qd").pack
_APPEND_ARGS = struct.Struct("@8P16q").pack

_HALF = {torch.bfloat16: _cabi.BF16, torch.float16: _cabi.FP16}
# The ops below are called once or more a layer for a single token, where a microsecond of checks is a tenth of the call: what a good call
# looks like is one expression, and the checks that name what is wrong run for the others.


def _check_w4a16(x, w_packed, w_scale, rows, per_channel) -> None:
    _half_input(x, "input", 2)
    K = x.shape[1]
    if per_channel:
        _require(K > 0 and K % 64 == 0, "K must be a multiple of 64")
    else:
        _require(K > 0 and K % 128 == 0, "K must be divisible by group_size")
    _require(w_packed.device == x.device and w_scale.device == x.device, "all tensors must be on the same device")
    _require(w_packed.dtype == torch.uint8 and w_packed.is_contiguous(), "b_packed must be contiguous uint8")
    _require(w_packed.numel() == rows * (K // 2), "b_packed does not have rows*K/2 bytes")
    _require(w_scale.dtype == torch.float32 and w_scale.is_contiguous(), "scale_b must be contiguous float32")
    _require(w_scale.numel() == (rows if per_channel else K // 128 * rows), "scale_b does not have a scale for every row (and group)")
    raise RuntimeError("w4a16_linear: unsupported arguments")


def _w4a16(x: torch.Tensor, w_packed: torch.Tensor, w_scale: torch.Tensor, N: int, per_channel: bool, gated: bool, who: str) -> torch.Tensor:
    rows = 2 * N if gated else N
    code = _HALF.get(x.dtype)
    if code is None or x.dim() != 2:
        _check_w4a16(x, w_packed, w_scale, rows, per_channel)
    M, K = x.shape
    index = x.get_device()
    if not (index >= 0 and K > 0 and K % (64 if per_channel else 128) == 0 and w_packed.get_device() == index and w_scale.get_device() == index
            and w_packed.dtype is torch.uint8 and w_scale.dtype is torch.float32 and w_packed.is_contiguous() and w_scale.is_contiguous()
            and w_packed.numel() * 2 == rows * K and w_scale.numel() == (rows if per_channel else K // 128 * rows)
            and not (x.requires_grad and torch.is_grad_enabled())):
        _check_w4a16(x, w_packed, w_scale, rows, per_channel)
    at = x.data_ptr()
    ldx, inner = x.stride()
    if M <= 1:
        ldx = K
    if inner != 1 or ldx % 8 or at % 16:
        x, ldx = x.clone(memory_format=torch.contiguous_format), K
        at = x.data_ptr()
    out = x.new_empty((M, N))
    args = _W4A16_ARGS(at, w_packed.data_ptr(), w_scale.data_ptr(), out.data_ptr(), code, M, K, ldx, N, per_channel, gated)
    rc = lib.i4tc_w4a16_linear(args, index, _raw_stream(index) if _raw_stream is not None else _stream(x))
    if rc:
        check(rc, who)
    return out


def w4a16_linear(x: torch.Tensor, w_packed: torch.Tensor, w_scale: torch.Tensor, N: int, per_channel: bool = False) -> torch.Tensor:
    """``x`` [M,K] (bf16 / fp16) times the transposed int4 weights of ``linear`` (codes [G,N,64] with scales [G,N], or [N,K/2] with [N]),
    without quantising the activations: exact products, fp32 sums, one rounding to ``x``'s type.  [M,N].  Made for the tokens of
    decoding: the weights are read once for every 32 of them."""
    return _w4a16(x, w_packed, w_scale, N, per_channel, False, "w4a16_linear")


def w4a16_gated_linear(x: torch.Tensor, w_packed: torch.Tensor, w_scale: torch.Tensor, inter: int, per_channel: bool = False) -> torch.Tensor:
    """``silu(x Wg^T) * (x Wu^T)`` [M,inter] in one kernel: ``w4a16_linear`` over fused gate and up weights (2 * inter rows, gate
    rows first, as ``moe_silu_mul_quant`` takes their product), with neither projection rounded before SwiGLU."""
    return _w4a16(x, w_packed, w_scale, inter, per_channel, True, "w4a16_gated_linear")


def rope_frequencies(rotary_dim: int, theta: float, device="cuda", scaling: str | None = None, factor: float = 1.0,
                     trained_length: int | None = None):
    """(frequencies float64 [rotary_dim / 2] in radians a position, scale of the rotated values) for ``rope``.

    ``scaling`` stretches a context ``factor`` times: ``"linear"`` divides all positions; ``"base"`` raises ``theta`` so that the slowest
    pair is stretched and the fastest stays; ``"by_parts"`` stretches the pairs that turn less than once within
    ``trained_length``, keeps those that turn more than 32 times, blends in between, and scales values by ``1 + ln(factor) / 10``."""
    _require(rotary_dim > 0 and rotary_dim % 2 == 0, "rotary_dim must be a positive even number")
    _require(scaling in (None, "linear", "base", "by_parts"), "scaling must be None, 'linear', 'base' or 'by_parts'")
    _require(theta > 0 and factor > 0, "theta and factor must be positive")
    if scaling == "base":
        _require(rotary_dim > 2, "scaling by the base needs more than one pair")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    freqs = [theta ** (-i / rotary_dim) for i in range(0, rotary_dim, 2)]
    scale = 1.0
    if scaling == "linear":
        freqs = [f / factor for f in freqs]
    elif scaling == "by_parts":
        _require(trained_length is not None and trained_length > 0, "scaling by parts needs trained_length")
        keep = [min(1.0, max(0.0, (trained_length * f / (2 * math.pi) - 1) / 31)) for f in freqs]
        freqs = [f * k + f / factor * (1 - k) for f, k in zip(freqs, keep)]
        scale = 1.0 + 0.1 * math.log(factor) if factor > 1 else 1.0
    return torch.tensor(freqs, dtype=torch.float64, device=device), scale


def _check_rope(x, positions, freqs) -> None:
    _half_input(x, "x", 3)
    tokens, _, D = x.shape
    _require(positions.dim() == 1 and positions.numel() == tokens, "positions must be [tokens]")
    _require(positions.dtype == torch.int64 or positions.dtype == torch.int32, "positions must be int32 or int64")
    _require(freqs.dtype == torch.float64 and freqs.dim() == 1 and freqs.is_contiguous(), "freqs must be a contiguous 1D float64 tensor")
    _require(2 * freqs.numel() <= D, "a head has fewer elements than the frequencies rotate")
    _require(positions.device == x.device and freqs.device == x.device, "all tensors must be on the same device")
    raise RuntimeError("rope: unsupported arguments")


def _rope(x, positions, freqs, interleaved, scale, inverse, in_place, who):
    code = _HALF.get(x.dtype)
    if code is None or x.dim() != 3:
        _check_rope(x, positions, freqs)
    tokens, heads, D = x.shape
    index, kind, R = x.get_device(), positions.dtype, 2 * freqs.numel()
    if not (index >= 0 and positions.get_device() == index and freqs.get_device() == index and positions.dim() == 1 and positions.numel() == tokens
            and (kind is torch.int64 or kind is torch.int32) and freqs.dtype is torch.float64 and freqs.dim() == 1 and freqs.is_contiguous()
            and R <= D and not (x.requires_grad and torch.is_grad_enabled())):
        _check_rope(x, positions, freqs)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    st, sh, sd = x.stride()
    if in_place:
        _require(sd == 1 or D <= 1, "elements of a head must be contiguous")
        (near, n), (far, m) = sorted(((sh, heads), (st, tokens)), key=lambda a: (a[1] > 1, a[0]))
        ok = (n <= 1 or near >= D) and (m <= 1 or far >= (near * (n - 1) if n > 1 else 0) + D)
        _require(ok or x.numel() == 0, "x overlaps itself")
        out, ot, oh = x, st, sh
    else:
        if sd != 1 and D > 1:
            x = x.contiguous()
            st, sh, sd = x.stride()
        out = x.new_empty((tokens, heads, D))
        ot, oh = heads * D, D
    if out.numel() == 0:
        return out
    # the stride of an axis of one counts for nothing
    if tokens == 1:
        st = ot = heads * D
    if heads == 1:
        sh = oh = D
    args = _ROPE_ARGS(x.data_ptr(), positions.data_ptr(), freqs.data_ptr(), out.data_ptr(), code, tokens, heads, D, R, st, sh, ot, oh,
                      kind is torch.int64, interleaved, inverse, scale)
    rc = lib.i4tc_rope(args, index, _raw_stream(index) if _raw_stream is not None else _stream(x))
    if rc:
        check(rc, who)
    return out


def rope(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool = False, scale: float = 1.0,
         inverse: bool = False) -> torch.Tensor:
    """Rotary embedding of ``x`` [tokens, heads, D] (bf16 / fp16, any strides) at ``positions`` [tokens] (int32 / int64): the first
    ``2 * len(freqs)`` elements of every head turn by ``position * freqs`` (float64, of ``rope_frequencies``) and are multiplied by
    ``scale``, the rest is copied.  Pairs are ``(i, i + R/2)``, or ``(2i, 2i + 1)`` with ``interleaved``.  ``inverse`` turns back: it moves
    keys to other positions, and is the gradient of ``rope``.  Angles are computed in 64 bits, so that they are good to fp32 at any int32
    position; one rounding.  Returns a new
    contiguous tensor."""
    return _rope(x, positions, freqs, interleaved, scale, inverse, False, "rope")


def rope_(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool = False, scale: float = 1.0,
          inverse: bool = False) -> torch.Tensor:
    """``rope`` in place, for instance on the query and key heads of a fused QKV buffer (``qkv.view(tokens, -1, D)[:, :heads]``)."""
    return _rope(x, positions, freqs, interleaved, scale, inverse, True, "rope_")


def _check_cache(k_cache, v_cache, block_table, lengths, k, v) -> None:
    for t, name in ((k, "k"), (v, "v"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _half_input(t, name, 4)
    _require(k.shape == v.shape, "k and v must have the same shape")
    _require(k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride(), "k_cache and v_cache must have the same shape and strides")
    _require(k.dtype == v.dtype == k_cache.dtype == v_cache.dtype, "keys, values and cache must have the same dtype")
    _require(k_cache.shape[2:] == k.shape[2:], "k_cache must be [pages, page_size, kv_heads, D] with the new keys' kv_heads and D")
    _require(k_cache.shape[1] > 0, "a page must hold at least one token")
    _require(k_cache.stride(3) == 1 or k.shape[3] <= 1, "elements of a cached head must be contiguous")
    B = k.shape[0]
    _require(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B, "block_table must be int32 [batch, pages of a sequence]")
    _require(lengths.dtype == torch.int32 and lengths.dim() == 1 and lengths.shape[0] == B, "lengths must be int32 [batch]")
    dev = k.device
    _require(v.device == dev and k_cache.device == dev and v_cache.device == dev and block_table.device == dev and lengths.device == dev,
             "all tensors must be on the same device")
    raise RuntimeError("unsupported arguments")


def _cache_pair(k_cache, v_cache, block_table, lengths, k, v):
    """Checks of a paged cache and the new rows beside it: (k, v, their strides, the cache's strides, block_table, lengths, device index, the sizes
    B, T, kv_heads, D, pages, page size, width of the table), k and v with the same strides."""
    kind, index = k.dtype, k.get_device()
    if not (kind in _HALF and index >= 0 and k.dim() == 4 and k_cache.dim() == 4 and block_table.dim() == 2 and lengths.dim() == 1):
        _check_cache(k_cache, v_cache, block_table, lengths, k, v)
    B, T, H, D = shape = k.shape
    pages, page, cache_heads, cache_D = cache_shape = k_cache.shape
    rows, width = block_table.shape
    new, cache = k.stride(), k_cache.stride()
    if not (v.dtype is kind and k_cache.dtype is kind and v_cache.dtype is kind and v.shape == shape and v_cache.shape == cache_shape
            and v_cache.stride() == cache and H == cache_heads and D == cache_D and page > 0 and (cache[3] == 1 or D <= 1)
            and block_table.dtype is torch.int32 and lengths.dtype is torch.int32 and rows == B and lengths.shape[0] == B
            and v.get_device() == index and k_cache.get_device() == index and v_cache.get_device() == index
            and block_table.get_device() == index and lengths.get_device() == index
            and not ((k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad) and torch.is_grad_enabled())):
        _check_cache(k_cache, v_cache, block_table, lengths, k, v)
    if v.stride() != new or new[3] != 1:
        k, v = k.contiguous(), v.contiguous()
        new = k.stride()
        if v.stride() != new:   # axes of one element: any stride counts as contiguous
            v = v.as_strided(shape, new)
    if block_table.stride(1) != 1 and width > 1:
        block_table = block_table.contiguous()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    return k, v, new, cache, block_table, lengths, index, (B, T, H, D, pages, page, width)


def kv_cache_append_(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor,
                     lengths: torch.Tensor, select: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> None:
    """Writes new keys and values [B, T, kv_heads, D] into a paged cache [pages, page_size, kv_heads, D] (keys and values each, same
    strides): row ``i < counts[b]`` (all T without ``counts``) becomes token ``lengths[b] + i`` of its sequence, in page
    ``block_table[b, token // page_size]``, and comes from new row ``select[b, i]`` (``i`` without ``select``): a prompt, or the accepted path
    of a tree of drafts.  All index tensors int32.  ``lengths`` stay as they are.  Counts, rows, tokens and pages out of range
    write nothing and are raised by ``check_status``.  No two rows may go to one place, and none to a place that ``k`` and ``v`` are read from
    (rows of the cache itself may be copied to other places of it)."""
    k, v, new, cache, block_table, lengths, index, sizes = _cache_pair(k_cache, v_cache, block_table, lengths, k, v)
    B, T = sizes[:2]
    counts_at = select_at = select_stride = 0
    if counts is not None:
        _require(counts.dtype is torch.int32 and counts.dim() == 1 and counts.shape[0] == B and counts.get_device() == index, "counts must be int32 [batch]")
        if not counts.is_contiguous():
            counts = counts.contiguous()
        counts_at = counts.data_ptr()
    if select is not None:
        _require(select.dtype is torch.int32 and select.dim() == 2 and select.shape[0] == B and select.get_device() == index,
                 "select must be int32 [batch, new rows]")
        _require(select.shape[1] >= T, "select must have as many columns as there are new rows")
        if select.stride(1) != 1:
            select = select.contiguous()
        select_at, select_stride = select.data_ptr(), select.stride(0)
    args = _APPEND_ARGS(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), lengths.data_ptr(),
                        counts_at, select_at, 2, *sizes, new[0], new[1], new[2], cache[0], cache[1], cache[2], block_table.stride(0), select_stride)
    rc = lib.i4tc_kv_append(args, index, _raw_stream(index) if _raw_stream is not None else _stream(k))
    if rc:
        check(rc, "kv_cache_append_")


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, lengths: torch.Tensor, tree_mask: torch.Tensor | None = None,
                   scale: float | None = None) -> torch.Tensor:
    """Attention of a few new tokens (up to 64: one, a chain, or a tree of drafts) over the cache of their sequence and one another.

    ``q`` [B, T, heads, D], ``k`` and ``v`` [B, T, kv_heads, D] are the new tokens' (any strides; not yet in the cache), ``heads`` a multiple of
    ``kv_heads``, D a multiple of 8 up to 128, bf16 / fp16.  The cache is that of ``kv_cache_append_``; token t sees its sequence's
    ``lengths[b]`` cached tokens and the new tokens j with ``tree_mask[b, t, j]`` (bool [B, T, T] or [T, T]; without one ``j <= t``).
    A token that sees nothing gives zeros, and what a token does not see has no part in its result, infinities and NaN
    included.  ``scale`` defaults to D ** -0.5.  Scores, weights' sums and results are held in fp32; a weight is rounded to the
    values' type before it multiplies them, as the tensor cores take it, and summed as rounded.  Returns [B, T, heads, D].  Pages
    and lengths out of range are raised by ``check_status``; the result of such a sequence means nothing, the others' stand."""
    kind = q.dtype
    code = _HALF.get(kind)
    if code is None or q.dim() != 4 or q.get_device() < 0 or (q.requires_grad and torch.is_grad_enabled()):
        _half_input(q, "q", 4)
    k, v, new, cache, block_table, lengths, index, (Bk, Tk, Hk, Dk, pages, page, width) = _cache_pair(k_cache, v_cache, block_table, lengths, k, v)
    B, T, H, D = q.shape
    if not (k.dtype is kind and q.get_device() == index and Bk == B and Tk == T and Dk == D and T <= 64 and D % 8 == 0 and 0 < D <= 128
            and Hk > 0 and H % Hk == 0):
        _require(kind == k.dtype and q.device == k.device, "queries must have the keys' dtype and device")
        _require(k.shape == (B, T, Hk, D), "q must be [B, T, heads, D] and k [B, T, kv_heads, D]")
        _require(T <= 64, "at most 64 new tokens a sequence")
        _require(D % 8 == 0 and 0 < D <= 128, "heads must have a multiple of 8 and at most 128 elements")
        _require(False, "heads must be a multiple of kv_heads")
    out = q.new_empty((B, T, H, D))
    if out.numel() == 0:
        return out
    mask_at = mask_batch = 0
    if tree_mask is not None:
        _require(tree_mask.dtype is torch.bool and tree_mask.get_device() == index, "tree_mask must be bool, on the queries' device")
        mask_shape = tree_mask.shape
        _require(mask_shape == (B, T, T) or mask_shape == (T, T), "tree_mask must be [B, T, T] or [T, T]")
        if not tree_mask.is_contiguous():
            tree_mask = tree_mask.contiguous()
        mask_at, mask_batch = tree_mask.data_ptr(), T * T if len(mask_shape) == 3 else 0
    sq, q_at = q.stride(), q.data_ptr()
    if sq[3] != 1 or (sq[0] | sq[1] | sq[2]) % 2 or q_at % 4:
        q = q.clone(memory_format=torch.contiguous_format)
        sq, q_at = q.stride(), q.data_ptr()
    k_at, v_at, k_cache_at, v_cache_at = k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    if (new[0] | new[1] | new[2]) % 8 or (k_at | v_at) % 16:
        k, v = (t.clone(memory_format=torch.contiguous_format) for t in (k, v))
        new, k_at, v_at = k.stride(), k.data_ptr(), v.data_ptr()
    _require((k_cache_at | v_cache_at) % 16 == 0 and (cache[0] | cache[1] | cache[2]) % 8 == 0, "cached heads must be 16-byte aligned")
    nbytes = lib.i4tc_tree_attention_scratch_bytes(B, T, H, Hk, D, width * page, index)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    args = _ATTENTION_ARGS(q_at, k_at, v_at, k_cache_at, v_cache_at, block_table.data_ptr(), lengths.data_ptr(), mask_at, out.data_ptr(),
                                0 if scratch is None else scratch.data_ptr(), nbytes, code, B, T, H, Hk, D, pages, page, width, sq[0], sq[1], sq[2], new[0], new[1], new[2],
                                cache[0], cache[1], cache[2], block_table.stride(0), mask_batch, D ** -0.5 if scale is None else scale)
    rc = lib.i4tc_tree_attention(args, index, _raw_stream(index) if _raw_stream is not None else _stream(q))
    if rc:
        check(rc, "tree_attention")
    return out


def set_tuning(tile_n: int = 0, swap: int = -1) -> None:
    """Force the GEMM tile width / operand orientation (tests); ``set_tuning()`` restores automatic."""
    check(lib.i4tc_set_tuning(tile_n, swap), "set_tuning")


def set_split_k(splits: int = 0) -> None:
    """Force the number of K ranges of the small-M per-group GEMM (tests); 0 restores automatic."""
    check(lib.i4tc_set_split_k(splits), "set_split_k")


def set_cta_pairs(mode: int = -1) -> None:
    """Force (1) or forbid (0) 256 x 256 tiles on SM pairs for large dense GEMMs (tests); -1 restores automatic."""
    check(lib.i4tc_set_cta_pairs(mode), "set_cta_pairs")


def set_small_m_path(path: int = 0) -> None:
    """Test / tuning hook: 0 = automatic, 1 = CUDA-core kernel only, 2 = register-fed tensor-core kernel wherever it
    applies (1..32 tokens), 3 = always the tile kernel."""
    check(lib.i4tc_set_small_m_path(path), "set_small_m_path")


def set_epilogue_warps(warps: int = 0) -> None:
    """Force 8 or 16 epilogue warps per thread block of the tensor-core GEMM (tests); 0 restores automatic."""
    check(lib.i4tc_set_epilogue_warps(warps), "set_epilogue_warps")


def reserve_workspace(nbytes: int, device=None, stream=None) -> None:
    """Make the split-K workspace of (device, stream) at least ``nbytes`` large now, so that no small-M GEMM on that
    stream allocates later (call before capturing a CUDA graph).  Defaults: current device, its current stream."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    st = torch.cuda.current_stream(dev) if stream is None else stream
    check(lib.i4tc_reserve_workspace(dev, st.cuda_stream, int(nbytes)), "reserve_workspace")


def workspace_bytes(device=None, stream=None) -> int:
    """Current size of the split-K workspace of (device, stream); 0 if none was needed yet."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    st = torch.cuda.current_stream(dev) if stream is None else stream
    return int(lib.i4tc_workspace_bytes(dev, st.cuda_stream))


def check_status(device=None) -> None:
    """Raise if any kernel gave up on a bounded wait, or met a length, page or index out of range, since the last call
    (synchronises the stream)."""
    dev = torch.cuda.current_device() if device is None else torch.device(device).index
    check(lib.i4tc_check_status(dev, torch.cuda.current_stream(dev).cuda_stream), "check_status")
