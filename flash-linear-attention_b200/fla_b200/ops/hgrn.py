# -*- coding: utf-8 -*-
"""Element-wise gated linear recurrence (HGRN): h_t = exp(g_t) h_{t-1} + x_t per channel, o_t = h_t. Public names and
arguments follow fla/ops/hgrn/chunk.py (`chunk_hgrn`) and fla/ops/hgrn/fused_recurrent.py (`fused_recurrent_hgrn`); both are
differentiable in x, g and the initial state, and both take packed sequences. The kernels are in csrc/hgrn.cu."""
from typing import Optional, Tuple

import torch

from .. import _lib
from .._lib import _DTYPES
from ..utils import resolve_offsets


def _p(t):
    return None if t is None else t.data_ptr()


def _workspace(lib, ref):
    """(scratch from the current stream's allocator, its bytes); none where every sequence is walked by itself."""
    n = lib.flab_hgrn_workspace(*ref.shape)
    return (torch.empty(n, dtype=torch.uint8, device=ref.device) if n else None), n


def hgrn_fwd(x, g, h0, output_final_state, cu):
    """x, g `[B, T, D]` contiguous, h0 `[N, D]` fp32 or None, cu int32 / int64 `[N + 1]` on the device or None."""
    B, T, D = x.shape
    N = B if cu is None else cu.numel() - 1
    o = torch.empty_like(x)
    ht = torch.empty(N, D, dtype=torch.float32, device=x.device) if output_final_state else None
    if x.numel() == 0 or N == 0:  # no token: the states pass through
        o.zero_()
        if ht is not None:
            ht.zero_() if h0 is None else ht.copy_(h0)
        return o, ht
    lib = _lib.load()
    ws, n = _workspace(lib, x)
    with _lib.device_of(x):
        rc = lib.flab_hgrn_fwd(x.data_ptr(), g.data_ptr(), _p(h0), o.data_ptr(), _p(ht), _p(cu), cu is not None and cu.dtype == torch.int64, B, T, D, N,
                               _DTYPES[x.dtype], _p(ws), n, _lib.stream_of(x))
    _lib.finish("flab_hgrn_fwd", rc)
    return o, ht


def hgrn_bwd(g, o, h0, do, dht, want_dh0, cu):
    B, T, D = g.shape
    N = B if cu is None else cu.numel() - 1
    dx, dg = torch.empty_like(g), torch.empty_like(g)
    dh0 = torch.empty(N, D, dtype=torch.float32, device=g.device) if want_dh0 else None
    if g.numel() == 0 or N == 0:
        dx.zero_(), dg.zero_()
        if dh0 is not None:
            dh0.zero_() if dht is None else dh0.copy_(dht)
        return dx, dg, dh0
    lib = _lib.load()
    ws, n = _workspace(lib, g)
    with _lib.device_of(g):
        rc = lib.flab_hgrn_bwd(g.data_ptr(), o.data_ptr(), _p(h0), do.data_ptr(), _p(dht), dx.data_ptr(), dg.data_ptr(), _p(dh0), _p(cu),
                               cu is not None and cu.dtype == torch.int64, B, T, D, N, _DTYPES[g.dtype], _p(ws), n, _lib.stream_of(g))
    _lib.finish("flab_hgrn_bwd", rc)
    return dx, dg, dh0


def _backward(ctx, do, dht):
    g, o, h0, cu = _lib.saved(ctx)
    do = torch.zeros_like(g) if do is None else do.to(g.dtype).contiguous()
    dht = None if dht is None else dht.float().contiguous()
    dx, dg, dh0 = hgrn_bwd(g, o, h0, do, dht, ctx.needs_input_grad[2], cu)
    return dx, dg, None if dh0 is None else dh0.to(ctx.h0_dtype), None, None


class HGRNFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, g, initial_state, output_final_state, cu):
        x, g = x.contiguous(), g.contiguous()
        h0 = None if initial_state is None else initial_state.detach().float().contiguous()
        o, ht = hgrn_fwd(x, g, h0, output_final_state, cu)
        ctx.save_for_backward(g, o, h0, cu)
        ctx.h0_dtype = None if initial_state is None else initial_state.dtype
        ctx.set_materialize_grads(False)
        return o, ht

    @staticmethod
    def backward(ctx, do, dht):
        return _lib.once(_backward)(ctx, do, dht)


def _hgrn(x, g, initial_state, output_final_state, offsets):
    if x.dim() != 3 or g.shape != x.shape:
        raise ValueError(f"x and g must both be [B, T, D], got {tuple(x.shape)} and {tuple(g.shape)}")
    if x.dtype not in _DTYPES or g.dtype != x.dtype:
        raise ValueError(f"x and g must share one of the types bfloat16, float16 and float32, got {x.dtype} and {g.dtype}")
    if max(x.shape[0], x.shape[2]) > 2 ** 30:  # (the C ABI takes them as ints)
        raise ValueError(f"x {tuple(x.shape)} has more than 2^30 sequences or channels, which the kernels do not index")
    if not x.is_cuda:
        raise RuntimeError("flab200 kernels run on CUDA tensors only (no CPU fallback)")
    N = x.shape[0]
    if offsets is not None:
        if x.shape[0] != 1:
            raise ValueError(f"The batch size is expected to be 1 rather than {x.shape[0]} when using `offsets`. "
                             f"Please flatten variable-length inputs before processing.")
        if offsets.dim() != 1 or offsets.dtype not in (torch.int32, torch.int64) or offsets.numel() < 1:
            raise ValueError(f"`offsets` must be a one-dimensional int32 or int64 tensor, got {offsets.dtype} {tuple(offsets.shape)}")
        offsets = offsets.to(x.device).contiguous()
        N = offsets.numel() - 1
    if g.device != x.device:
        raise RuntimeError(f"g is on {g.device}, expected {x.device}")
    if initial_state is not None and initial_state.device != x.device:
        raise RuntimeError(f"initial_state is on {initial_state.device}, expected {x.device}")
    if initial_state is not None and tuple(initial_state.shape) != (N, x.shape[2]):
        raise ValueError(f"The number of initial states is expected to be equal to the number of input sequences, "
                         f"i.e., a shape of {(N, x.shape[2])} rather than {tuple(initial_state.shape)}.")
    if (torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or (initial_state is not None and initial_state.requires_grad))) \
            or _lib.dual(x, g, initial_state):
        return HGRNFunction.apply(x, g, initial_state, bool(output_final_state), offsets)
    h0 = None if initial_state is None else initial_state.float().contiguous()
    return hgrn_fwd(x.contiguous(), g.contiguous(), h0, bool(output_final_state), offsets)


def chunk_hgrn(
    x: torch.Tensor,
    g: torch.Tensor,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    offsets: Optional[torch.LongTensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """h_t = exp(g_t) h_{t-1} + x_t along dim 1, element by element.

    x, g: `[B, T, D]` of one type (bf16, fp16 or fp32), g the log of the forget gate; initial_state `[N, D]` or None (zeros).
    offsets (or `cu_seqlens`): int32 / int64 `[N + 1]` cumulative lengths of N sequences packed into B = 1, non-decreasing
    and within [0, T]. They are read on the device only (no synchronisation, so a call can be captured into a CUDA graph); a
    sequence may be empty, and tokens outside every sequence get zeros in o and in the gradients.
    Returns (o `[B, T, D]`, final_state `[N, D]` fp32 or None)."""
    return _hgrn(x, g, initial_state, output_final_state, resolve_offsets(offsets, cu_seqlens))


def fused_recurrent_hgrn(
    x: torch.Tensor,
    g: torch.Tensor,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    offsets: Optional[torch.LongTensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The same recurrence under the name that decode loops call (one or a few tokens a step; arguments as `chunk_hgrn`)."""
    return _hgrn(x, g, initial_state, output_final_state, resolve_offsets(offsets, cu_seqlens))
