"""Products of 8-bit floating point values (e4m3) with one fp32 scale for each block of 128 along the reduction.

Activations and incoming gradients have a scale for each row and 128 columns, weights one for each 128 x 128 values.  The
tensor cores add up each block by itself; the block's two scales multiply it in fp32 before it joins the others
(``csrc/fp8.cu``).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import backward_follows, cpp_nodes, functional as Fn, native, use_native

MAX_SIZE = 2 ** 31 - 256         # rows and columns, which the kernels round up to whole tiles in 32 bits


def _check_size(name: str, x) -> None:
    if max(x.shape) > MAX_SIZE:
        raise ValueError(f"{name} {list(x.shape)} has more than 2^31 - 256 rows or columns")


def quantize_fp8(x: torch.Tensor, block_rows: int = 1):
    """``(values e4m3 [M, K], scales fp32)`` of ``x [M, K]`` (fp32, bf16 or fp16).  ``block_rows`` 1: a scale for each row and
    128 columns, ``[M, ceil(K / 128)]``; 128: one for each 128 x 128 values, ``[ceil(M / 128), ceil(K / 128)]``.  A scale is
    ``max(largest / 448, 2^-120)``, a value ``x / scale`` rounded to nearest.  On a GPU the rows of the values start at
    multiples of 16 bytes, as ``matmul_fp8`` reads them.  NaN stays NaN; a block with an infinity has an infinite scale."""
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [rows, columns] with a column at least, got {list(x.shape)}")
    _check_size("x", x)
    if block_rows not in (1, 128):
        raise ValueError(f"block_rows must be 1 or 128, got {block_rows}")
    if not x.dtype.is_floating_point:
        raise TypeError(f"x must be floating point, got {x.dtype}")
    if not use_native(x, "fp8"):
        return Fn.quantize_fp8_ref(x, block_rows)
    return native.quantize_fp8(x.detach() if x.stride(1) == 1 else x.detach().contiguous(), block_rows)


def _check_operand(name: str, values, scales, block_rows: int) -> None:
    if values.dim() != 2 or min(values.shape[1], 1) < 1 or values.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{name} must be float8_e4m3fn [rows, columns], got {values.dtype} {list(values.shape)}")
    _check_size(name, values)
    want = ((values.shape[0] + block_rows - 1) // block_rows, (values.shape[1] + 127) // 128)
    if scales.dtype != torch.float32 or tuple(scales.shape) != want or scales.device != values.device:
        raise ValueError(f"the scales of {name} {list(values.shape)} must be fp32 {list(want)} on {values.device}, got "
                         f"{scales.dtype} {list(scales.shape)} on {scales.device}")


def _rows_aligned(name: str, values) -> None:
    """What a tensor map takes."""
    if values.stride(1) != 1 or values.stride(0) % 16 or values.data_ptr() % 16 or values.stride(0) < values.shape[1]:
        raise ValueError(f"the rows of {name} must be contiguous and start at multiples of 16 bytes (as quantize_fp8 returns "
                         f"them), got strides {values.stride()}")


def matmul_fp8(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor) -> torch.Tensor:
    """``a [M, K] @ b [N, K]ᵀ`` as bf16 ``[M, N]``: e4m3 values, ``a_scales [M, ceil(K / 128)]``, ``b_scales [ceil(N / 128),
    ceil(K / 128)]`` (any strides).  Sums are held in fp32.  It has no gradient of its own; ``linear_fp8`` has."""
    if use_native(a, "fp8"):
        nodes = cpp_nodes(a, a_scales, b, b_scales)
        out = nodes.matmul_fp8(a, a_scales, b, b_scales, native.status_word(a.device)) if nodes else None
        if out is not None:
            return out
    _check_operand("a", a, a_scales, 1)
    _check_operand("b", b, b_scales, 128)
    if a.shape[1] != b.shape[1] or a.device != b.device:
        raise ValueError(f"a {list(a.shape)} on {a.device} and b {list(b.shape)} on {b.device} must share K and the device")
    if not use_native(a, "fp8"):
        return (Fn.dequantize_fp8_ref(a, a_scales, 1) @ Fn.dequantize_fp8_ref(b, b_scales, 128).t()).to(torch.bfloat16)
    if b.shape[0] == 0:
        return torch.empty(a.shape[0], 0, dtype=torch.bfloat16, device=a.device)
    _rows_aligned("a", a)
    _rows_aligned("b", b)
    return native.gemm_fp8(a, a_scales, b, b_scales)


def _product(x, values, scales, transposed: bool):
    """``x`` quantised by rows, times the weight (``transposed``) or along its rows."""
    if use_native(x, "fp8"):
        return native.gemm_fp8(*native.quantize_fp8(x, 1), values, scales, nn=not transposed)
    weight = Fn.dequantize_fp8_ref(values, scales, 128)
    return (Fn.dequantize_fp8_ref(*Fn.quantize_fp8_ref(x, 1), 1) @ (weight.t() if transposed else weight)).to(x.dtype)


def _aligned_rows(t):
    """``t [M, K]`` itself, or a copy where a tensor map does not take its rows."""
    if t.stride(1) == 1 and t.stride(0) * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0 and t.stride(0) >= t.shape[1]:
        return t
    return t.clone(memory_format=torch.contiguous_format)


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, values, scales):
        x2d = _aligned_rows(x.reshape(-1, x.shape[-1]))
        y = _product(x2d, values, scales, True)
        ctx.weight = weight
        ctx.save_for_backward(x2d, values, scales)
        ctx.shape = x.shape
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2d, values, scales = ctx.saved_tensors
        weight = ctx.weight
        dy2d = _aligned_rows(dy.reshape(-1, dy.shape[-1]))
        dx = _product(dy2d, values, scales, False).view(ctx.shape) if ctx.needs_input_grad[0] else None
        main_grad = getattr(weight, "main_grad", None)
        dw = None
        on_gpu = use_native(dy2d, "gemm") and dy2d.shape[0] > 0       # no rows: zeros
        if main_grad is not None:
            if on_gpu:
                native.gemm_tn(dy2d, x2d, out=main_grad, accumulate=True)
            else:
                main_grad.addmm_(dy2d.t().to(main_grad.dtype), x2d.to(main_grad.dtype))
        elif ctx.needs_input_grad[1]:
            dw = native.gemm_tn(dy2d, x2d, out_dtype=weight.dtype) if on_gpu else \
                (dy2d.float().t() @ x2d.float()).to(weight.dtype)
        return dx, dw, None, None


def linear_fp8(x: torch.Tensor, weight: torch.Tensor, weight_fp8=None) -> torch.Tensor:
    """``y = x @ weightᵀ`` with both operands in 8-bit floating point: ``x [..., d_in]`` (bf16) is quantised by rows of 128,
    ``weight [d_out, d_in]`` by blocks of 128 x 128 or given so (``weight_fp8 = quantize_fp8(weight, 128)``, to be renewed
    when the weight changes).  The gradient of ``x`` is the same kind of product of ``dy``, quantised by rows of 128, with the
    same values of the weight; that of the weight is the bf16 product ``dyᵀ x``, added to ``weight.main_grad`` where there is
    one, like ``linear``'s."""
    if use_native(x, "fp8") and getattr(weight, "pending_gather", None) is None:
        values, scales = (None, None) if weight_fp8 is None else weight_fp8
        nodes = cpp_nodes(x, weight, *(() if values is None else (values, scales)))
        out = nodes.linear_fp8(x, weight, values, scales, native.status_word(x.device)) if nodes else None
        if out is not None:
            return out
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or min(weight.shape) < 1:
        raise ValueError(f"x {list(x.shape)} and weight {list(weight.shape)} must share their last dimension, and the weight have a row")
    _check_size("weight", weight)
    if x.numel() // x.shape[-1] > MAX_SIZE:
        raise ValueError(f"x {list(x.shape)} has more than 2^31 - 256 rows")
    if x.device != weight.device:
        raise ValueError(f"x is on {x.device}, the weight on {weight.device}")
    if getattr(weight, "pending_gather", None) is not None:
        raise ValueError("the weight is still to be gathered")
    on_gpu = use_native(x, "fp8")
    if on_gpu and x.dtype != torch.bfloat16:
        raise TypeError(f"x must be bfloat16, got {x.dtype}")
    follows = backward_follows(x, weight)
    if on_gpu and follows and (weight.requires_grad or getattr(weight, "main_grad", None) is not None):
        # what the bf16 product of the weight gradient takes
        if weight.shape[0] % 8 or weight.shape[1] % 32 or weight.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("the weight gradient needs a bf16 or fp32 weight with d_out a multiple of 8 and d_in one of 32, got "
                             f"{weight.dtype} {list(weight.shape)}")
    if weight_fp8 is None:
        weight_fp8 = quantize_fp8(weight.detach(), 128)
    else:
        _check_operand("weight_fp8", *weight_fp8, 128)
        if weight_fp8[0].shape != weight.shape or weight_fp8[0].device != x.device:
            raise ValueError(f"weight_fp8 {list(weight_fp8[0].shape)} does not fit the weight {list(weight.shape)}")
        if on_gpu:
            _rows_aligned("weight_fp8", weight_fp8[0])
    return _LinearFp8.apply(x, weight, *weight_fp8)
