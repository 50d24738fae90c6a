# -*- coding: utf-8 -*-
"""RMS norm with the residual's addition, with the names of fla/modules/layernorm.py (`rms_norm`, `RMSNorm`), and its form with an
8-bit output for `linear_fp8` (`rms_norm_quant`; `quantize_rows` is the same output without the norm). The kernels are in
csrc/rms_norm.cu. A weight, no bias; mean subtraction and a bias are not built."""
import math
from typing import Optional

import torch
import torch.nn as nn

from .. import _lib
from .._lib import _DTYPES

NORM_E4M3, NORM_NONE = 1, 2


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(x: torch.Tensor) -> torch.Tensor:
    if x.dim() == 2:
        return x.contiguous()
    return x.reshape(math.prod(x.shape[:-1]), x.shape[-1]).contiguous()


def _like(t: torch.Tensor, shape) -> torch.Tensor:
    return t if t.shape == shape else t.reshape(shape)


def _forward(x, w, r, eps, sum_dtype, want_sum, want_rstd, quant=False, norm=True):
    """Returns (y, scale, sum, rstd), None for what was not asked for; y and sum have x's shape from the start, so that outputs of an
    autograd Function are no views and may be changed in place."""
    x2, r2 = _rows(x), None if r is None else _rows(r)
    w = None if w is None else w.contiguous()
    rows, n = x2.shape
    flat = dict(memory_format=torch.contiguous_format)  # (empty() from sizes takes 1 us longer)
    y = torch.empty_like(x, dtype=torch.float8_e4m3fn, **flat) if quant else torch.empty_like(x, **flat)
    total = torch.empty_like(x, dtype=sum_dtype, **flat) if want_sum else None
    rstd = x2.new_empty(rows, dtype=torch.float32) if want_rstd else None
    scale = x2.new_empty(rows, dtype=torch.float32) if quant else None
    if rows and n:
        lib = _lib.load()
        with _lib.device_of(x2):
            rc = lib.flab_rms_norm_fwd(x2.data_ptr(), _p(r2), _p(w), y.data_ptr(), _p(total), _p(rstd), _p(scale), rows, n, _DTYPES[x2.dtype],
                                       _DTYPES[x2.dtype if r2 is None else r2.dtype], _DTYPES[sum_dtype],
                                       _DTYPES[torch.float32 if w is None else w.dtype], NORM_E4M3 * quant + NORM_NONE * (not norm), eps,
                                       _lib.stream_of(x2))
        _lib.finish("flab_rms_norm_fwd", rc)
    elif quant:
        scale.zero_()  # rows of no elements
    return y, scale, total, rstd


def _backward(ctx, dy, dsum=None):
    total, rstd, w = _lib.saved(ctx)
    total = _rows(total)
    rows, n = total.shape
    need_x, need_w, need_r = ctx.needs_input_grad[:3]
    dy = torch.zeros_like(total, dtype=ctx.x_dtype) if dy is None else _rows(dy if dy.dtype == ctx.x_dtype else dy.to(ctx.x_dtype))
    dsum = None if dsum is None else _rows(dsum if dsum.dtype == total.dtype else dsum.to(total.dtype))
    wide = need_r and ctx.r_dtype != ctx.x_dtype  # the residual's gradient has a type of its own (the sum's)
    dx = torch.empty_like(dy) if need_x or (need_r and not wide) else None
    dr = torch.empty_like(total) if wide else None
    dw = torch.empty_like(w) if w is not None and need_w else None
    if rows and n:
        lib = _lib.load()
        part = None
        with _lib.device_of(total):
            if dw is not None:
                part = rstd.new_empty((lib.flab_rms_norm_partials(rows, n, _DTYPES[ctx.x_dtype]), n))
            rc = lib.flab_rms_norm_bwd(total.data_ptr(), dy.data_ptr(), _p(dsum), _p(w), rstd.data_ptr(), _p(dx), _p(dr), _p(dw), _p(part),
                                       rows, n, _DTYPES[ctx.x_dtype], _DTYPES[total.dtype],
                                       _DTYPES[torch.float32 if w is None else w.dtype], _lib.stream_of(total))
        _lib.finish("flab_rms_norm_bwd", rc)
    elif dw is not None:
        dw.zero_()
    dx = None if dx is None else _like(dx, ctx.x_shape)
    dr = _like(dr, ctx.x_shape) if wide else dx
    return dx if need_x else None, dw, dr if need_r else None, None, None, None


class RMSNormFunction(torch.autograd.Function):
    """(y, sum) or y alone; `sum` is x itself, and not among the outputs, where there is neither a residual nor a wider type."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps, sum_dtype, prenorm):
        w = None if weight is None else weight.contiguous()
        own_sum = residual is not None or sum_dtype != x.dtype
        x = x.contiguous()
        y, _, total, rstd = _forward(x, w, residual, eps, sum_dtype, own_sum, True)
        ctx.save_for_backward(total if own_sum else x, rstd, w)
        ctx.x_shape, ctx.x_dtype = x.shape, x.dtype
        ctx.r_dtype = None if residual is None else residual.dtype
        ctx.set_materialize_grads(False)
        return (y, total) if prenorm else y

    @staticmethod
    def backward(ctx, dy, dsum=None):
        return _lib.once(_backward)(ctx, dy, dsum)


def _check(x, weight, residual, residual_in_fp32):
    """The arguments' checks; returns the type of the residual stream."""
    if x.dim() < 1 or x.dtype not in _DTYPES:
        raise ValueError(f"x must be bfloat16, float16 or float32 with at least one dimension, got {x.dtype} {tuple(x.shape)}")
    if x.shape[-1] > 2 ** 30:  # (the C ABI takes it as an int)
        raise ValueError(f"rows of {x.shape[-1]} elements are beyond 2^30, which the kernels do not index")
    if weight is not None and (tuple(weight.shape) != (x.shape[-1],) or weight.dtype not in _DTYPES):
        raise ValueError(f"weight must be [{x.shape[-1]}] in bfloat16, float16 or float32, got {weight.dtype} {tuple(weight.shape)}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must have the shape of x, {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"residual must have the type of x ({x.dtype}) or float32, got {residual.dtype}")
    if not x.is_cuda:
        raise RuntimeError("flab200 kernels run on CUDA tensors only (no CPU fallback)")
    for name, t in (("weight", weight), ("residual", residual)):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{name} is on {t.device}, expected {x.device}")
    return torch.float32 if residual_in_fp32 else x.dtype if residual is None else residual.dtype


def _differentiable(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _refuse_derivatives(name, *tensors):
    if _differentiable(*tensors):
        raise NotImplementedError(f"{name} has no backward: call it under torch.no_grad()")
    if _lib.dual(*tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6, prenorm: bool = False, residual_in_fp32: bool = False):
    """y = s / sqrt(mean(s^2) + eps) * weight over the last dimension, s = x + residual.

    x `[..., n]` bf16, fp16 or fp32; weight `[n]` of any of these or None; residual of x's shape, in x's type or fp32. s is rounded to
    the type in which the residual stream is kept (fp32 with `residual_in_fp32`, else the residual's, else x's) and y is computed from
    the rounded s in fp32. Returns y in x's type, or with `prenorm` (y, s), both differentiable."""
    if bias is not None:
        raise NotImplementedError("rms_norm: a bias is not built")
    sum_dtype = _check(x, weight, residual, residual_in_fp32)
    same = residual is None and sum_dtype == x.dtype  # the stream is x
    if _differentiable(x, weight, residual) or _lib.dual(x, weight, residual):
        out = RMSNormFunction.apply(x, weight, residual, float(eps), sum_dtype, prenorm and not same)
        return (out, x) if prenorm and same else out
    y, _, total, _ = _forward(x, weight, residual, float(eps), sum_dtype, prenorm and not same, False)
    return (y, x if same else total) if prenorm else y


def rms_norm_quant(x: torch.Tensor, weight: Optional[torch.Tensor], residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   prenorm: bool = False, residual_in_fp32: bool = False):
    """`rms_norm` with an 8-bit output for `linear_fp8`: (q, scale) or, with `prenorm`, (q, scale, s).

    q `[..., n]` float8_e4m3fn and scale `[...]` fp32 stand for q * scale; scale is the row's largest |y| / 448, and 0 for a row of
    zeros. (Where that lies below fp32's normal numbers it is 2^-126 for 16-bit x, and rounded up for fp32 x.) For inference: there is no backward, and a call that would need one is refused."""
    sum_dtype = _check(x, weight, residual, residual_in_fp32)
    _refuse_derivatives("rms_norm_quant", x, weight, residual)
    same = residual is None and sum_dtype == x.dtype
    q, scale, total, _ = _forward(x, weight, residual, float(eps), sum_dtype, prenorm and not same, False, quant=True)
    scale = _like(scale, x.shape[:-1])
    return (q, scale, x if same else total) if prenorm else (q, scale)


def quantize_rows(x: torch.Tensor):
    """(q float8_e4m3fn of x's shape, scale fp32 of x's leading dimensions): x row by row as q * scale, scale = max|x| / 448. What
    `linear_fp8` takes for weights (`[N, K]`, one scale an output) and for tokens that do not come out of `rms_norm_quant`."""
    _check(x, None, None, False)
    _refuse_derivatives("quantize_rows", x)
    q, scale, _, _ = _forward(x, None, None, 0.0, x.dtype, False, False, quant=True, norm=False)
    return q, _like(scale, x.shape[:-1])


class RMSNorm(nn.Module):

    def __init__(self, hidden_size: int, elementwise_affine: bool = True, bias: bool = False, eps: float = 1e-5):
        super().__init__()
        if bias:
            raise NotImplementedError("RMSNorm: a bias is not built")
        self.hidden_size = hidden_size
        self.elementwise_affine = elementwise_affine
        self.eps = eps
        self.register_parameter("weight", nn.Parameter(torch.ones(hidden_size)) if elementwise_affine else None)
        self.register_parameter("bias", None)

    def __repr__(self) -> str:
        return f"{self.__class__.__name__}({self.hidden_size}, eps={self.eps})"

    def forward(self, x, residual=None, prenorm=False, residual_in_fp32=False):
        return rms_norm(x, self.weight, self.bias, residual=residual, eps=self.eps, prenorm=prenorm, residual_in_fp32=residual_in_fp32)
