# -*- coding: utf-8 -*-
"""Projections as one kernel each: a product with bias, activation and residual in its epilogue (`linear`), and the same for e4m3
tokens and weights with a scale a row (`linear_fp8`; `rms_norm_quant` and `quantize_rows` make them). They stand for nn.Linear and the
elementwise steps around it in fla/layers (gate and input projections in front of a recurrence, the output projection onto the
residual stream). The kernels are in csrc/linear.cu."""
import math
from typing import Optional

import torch

from .. import _lib
from .._lib import _DTYPES

ACTIVATIONS = {None: 0, "silu": 1, "swish": 1, "sigmoid": 2, "logsigmoid": 3, "gelu": 4}
_HALF = (torch.bfloat16, torch.float16)
_LARGEST = 2 ** 30  # rows or columns (the C ABI takes them as ints)


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(x: torch.Tensor) -> torch.Tensor:
    if x.dim() == 2:
        return x.contiguous()
    return x.reshape(math.prod(x.shape[:-1]), x.shape[-1]).contiguous()


def _like(t: torch.Tensor, shape) -> torch.Tensor:
    return t if t.shape == shape else t.reshape(shape)


def _as_is(t: torch.Tensor, n: int) -> bool:
    """Whether rows of n elements begin on 16-byte boundaries, as the kernel reads its operands."""
    return n % 8 == 0 and t.data_ptr() % 16 == 0


def _forward(x2, w, b, r2, act, want_z, lead):
    """(y, z or None, the operands' copies or None); y is [*lead, N] from the start, so that the output of an autograd Function is no
    view and may be changed in place."""
    (M, K), N = x2.shape, w.shape[0]
    y = torch.empty(*lead, N, dtype=x2.dtype, device=x2.device)
    z = torch.empty_like(y) if want_z else None
    copies = None
    if M:
        lib = _lib.load()
        n = 0 if _as_is(x2, K) and _as_is(w, K) else lib.flab_linear_workspace(x2.data_ptr(), w.data_ptr(), M, N, K)
        if n:
            copies = torch.empty(n, dtype=torch.uint8, device=x2.device)
        with _lib.device_of(x2):  # (the scratch's size goes by the device's)
            m = lib.flab_linear_scratch(M, N, K, _DTYPES[x2.dtype])
            scratch = torch.empty(m, dtype=torch.uint8, device=x2.device) if m else None
            rc = lib.flab_linear_fwd(x2.data_ptr(), w.data_ptr(), _p(b), _p(r2), y.data_ptr(), _p(z), M, N, K, act, _DTYPES[x2.dtype], _p(copies), n,
                                     _p(scratch), m, _lib.stream_of(x2))
        _lib.finish("flab_linear_fwd", rc)
    return y, z, copies


def _backward(ctx, dy):
    # (rows that began on 16-byte boundaries when they were saved do so again, and copies on one of 256 bytes)
    x2, w, z, copies = (t if t is None or t.data_ptr() % to == 0 else t.clone() for t, to in zip(_lib.saved(ctx), (16, 16, 1, 256)))
    need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    M, N, K = ctx.sizes
    d2, dev = _rows(dy), dy.device
    dx = torch.empty(M, K, dtype=dy.dtype, device=dev) if need_x else None
    dw = torch.empty(N, K, dtype=dy.dtype, device=dev) if need_w else None
    db = torch.empty(N, dtype=dy.dtype, device=dev) if need_b else None
    if M == 0:
        for t in (dw, db):
            if t is not None:
                t.zero_()
    elif need_x or need_w or need_b:
        lib = _lib.load()
        # Kept operands are read where they are now (a checkpoint or a hook may have brought them back elsewhere). One that was copied, or
        # whose product is not wanted, is not kept: its address in forward only says how the copies lie.
        x_at, w_at = (at if t is None else t.data_ptr() for t, at in zip((x2, w), ctx.places))
        with _lib.device_of(d2):
            n = lib.flab_linear_bwd_scratch(d2.data_ptr(), M, N, K, ctx.act) if need_x or need_w else 0
            scratch = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
            part = torch.empty(lib.flab_linear_bwd_partials(M, N), N, dtype=torch.float32, device=dev) if need_b else None
            rc = lib.flab_linear_bwd(x_at, w_at, _p(z), d2.data_ptr(), _p(dx), _p(dw), _p(db), _p(part), M, N, K, ctx.act, _DTYPES[dy.dtype],
                                     _p(copies), 0 if copies is None else copies.numel(), _p(scratch), n, _lib.stream_of(d2))
        _lib.finish("flab_linear_bwd", rc)
    return (None if dx is None else _like(dx, ctx.x_shape)), dw, db, (dy if need_r else None), None


class LinearFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x2, w = _rows(x), weight.contiguous()
        need_x, need_w, need_b, _ = ctx.needs_input_grad[:4]
        y, z, copies = _forward(x2, w, None if bias is None else bias.contiguous(), None if residual is None else _rows(residual), act,
                                act != 0 and (need_x or need_w or need_b), x.shape[:-1])
        K = w.shape[1]
        ctx.save_for_backward(x2 if need_w and _as_is(x2, K) else None, w if need_x and _as_is(w, K) else None, z, copies if need_x or need_w else None)
        ctx.places = x2.data_ptr(), w.data_ptr()
        ctx.act, ctx.sizes, ctx.x_shape = act, (x2.shape[0], w.shape[0], K), x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        return _lib.once(_backward)(ctx, dy)


def _check(x, weight, bias, residual, activation, dtype):
    if activation not in ACTIVATIONS:
        raise ValueError(f"Activation `{activation}` not supported: one of None, silu (swish), sigmoid, logsigmoid and gelu.")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"x must be [..., K] and weight [N, K] with N, K > 0, got {tuple(x.shape)} and {tuple(weight.shape)}")
    N = weight.shape[0]
    if max(math.prod(x.shape[:-1]), N, x.shape[-1]) > _LARGEST:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} have sides beyond 2^30, which the kernels do not index")
    if bias is not None and (tuple(bias.shape) != (N,) or bias.dtype != dtype):
        raise ValueError(f"bias must be [{N}] in {dtype}, got {bias.dtype} {tuple(bias.shape)}")
    if residual is not None and (residual.shape != x.shape[:-1] + (N,) or residual.dtype != dtype):
        raise ValueError(f"residual must be {tuple(x.shape[:-1]) + (N,)} in {dtype}, got {residual.dtype} {tuple(residual.shape)}")
    if not x.is_cuda:
        raise RuntimeError("flab200 kernels run on CUDA tensors only (no CPU fallback)")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.device != x.device:
            raise RuntimeError(f"{name} is on {t.device}, expected {x.device}")


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
           activation: Optional[str] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual, differentiable in all four tensors.

    x `[..., K]`, weight `[N, K]`, bias `[N]`, residual `[..., N]`, all of one type, bf16 or fp16 (fp32 is refused: the tensor
    cores would round it); activation None, "silu" (or "swish"), "sigmoid", "logsigmoid" (a log forget gate) or "gelu" (erf)."""
    if x.dtype not in _HALF or weight.dtype != x.dtype:
        raise ValueError(f"x and weight must both be bfloat16 or both float16, got {x.dtype} and {weight.dtype}")
    _check(x, weight, bias, residual, activation, x.dtype)
    act = ACTIVATIONS[activation]
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))) or _lib.dual(x, weight, bias, residual):
        return LinearFunction.apply(x, weight, bias, residual, act)
    return _forward(_rows(x), weight.contiguous(), None if bias is None else bias.contiguous(), None if residual is None else _rows(residual), act, False,
                    x.shape[:-1])[0]


def linear_fp8(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
               residual: Optional[torch.Tensor] = None, activation: Optional[str] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """act((x x_scale)(weight weight_scale)^T + bias) + residual for float8_e4m3fn x `[..., K]` and weight `[N, K]` with fp32 scales
    `[...]` and `[N]`, as `rms_norm_quant` and `quantize_rows` return them. K a multiple of 16; bias, residual and the result in
    out_dtype, bf16 or fp16. For inference: no backward."""
    e4m3 = torch.float8_e4m3fn
    if x.dtype != e4m3 or weight.dtype != e4m3 or out_dtype not in _HALF:
        raise ValueError(f"x and weight must be float8_e4m3fn and out_dtype bfloat16 or float16, got {x.dtype}, {weight.dtype} and {out_dtype}")
    for name, s, shape in (("x_scale", x_scale, x.shape[:-1]), ("weight_scale", weight_scale, weight.shape[:1])):
        if s.dtype != torch.float32 or s.shape != shape or s.device != x.device:
            raise ValueError(f"{name} must be {tuple(shape)} in float32 on {x.device}, got {s.dtype} {tuple(s.shape)} on {s.device}")
    _check(x, weight, bias, residual, activation, out_dtype)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, x_scale, weight, weight_scale, bias, residual)):
        raise NotImplementedError("linear_fp8 has no backward: call it under torch.no_grad()")
    if _lib.dual(x, x_scale, weight, weight_scale, bias, residual):
        raise NotImplementedError("linear_fp8 has no forward-mode derivative")
    if x.shape[-1] % 16:
        raise ValueError(f"linear_fp8: K = {x.shape[-1]} must be a multiple of 16")
    x2, w = _rows(x), weight.contiguous()
    if x2.data_ptr() % 16:
        x2 = x2.clone()
    if w.data_ptr() % 16:
        w = w.clone()
    b, r2 = None if bias is None else bias.contiguous(), None if residual is None else _rows(residual)
    xs, ws = x_scale.contiguous(), weight_scale.contiguous()
    (M, K), N = x2.shape, w.shape[0]
    y = torch.empty(*x.shape[:-1], N, dtype=out_dtype, device=x.device)
    if M:
        lib = _lib.load()
        with _lib.device_of(x2):
            n = lib.flab_linear_scratch(M, N, K, 3)
            scratch = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
            rc = lib.flab_linear_e4m3(x2.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), _p(b), _p(r2), y.data_ptr(), M, N, K,
                                      ACTIVATIONS[activation], _DTYPES[out_dtype], _p(scratch), n, _lib.stream_of(x2))
        _lib.finish("flab_linear_e4m3", rc)
    return y
