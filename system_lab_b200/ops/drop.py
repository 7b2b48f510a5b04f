"""Dropout from a counter-based generator (``csrc/dropout.cu``): the mask is a function of a seed, an offset and the
element's index in the (contiguous) tensor, so it is never stored; backward makes it again.

Calls that are to have different masks differ in ``seed`` or ``offset``: every offset is a stream of its own for tensors of
up to 2^67 elements.  ``seed`` may be an int64 tensor of one element on the tensor's device, read when the kernel runs, so
that a replayed graph draws the masks of the seed it finds there; its value at the time of the forward pass is kept for the
backward pass (a copy of eight bytes).
"""
from __future__ import annotations

import torch

from . import cuda
from . import reference as ref

cuda.register("slab_dropout", "pppililpls")

_TYPES = (torch.float32, torch.bfloat16)


def _signed(v: int) -> int:
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >> 63 else v


def check(x, p, seed, offset, residual):
    if not x.is_floating_point():
        raise ValueError(f"dropout of {x.dtype}")
    if not 0.0 <= p < 1.0 or ref.dropout_threshold(p) > 65535:
        raise ValueError(f"dropout probability {p}: has to be at least 0 and below 1 - 2^-17")
    if isinstance(seed, torch.Tensor):
        if seed.numel() != 1 or seed.dtype != torch.int64 or seed.device != x.device:
            raise ValueError("a seed in a tensor has to be one int64 on x's device")
    elif not isinstance(seed, int) or isinstance(seed, bool) or not -(1 << 63) <= seed < 1 << 64:
        raise ValueError(f"seed {seed!r}: has to be a 64-bit integer or an int64 tensor of one element")
    if not isinstance(offset, int) or isinstance(offset, bool) or not 0 <= offset < 1 << 64:
        raise ValueError(f"offset {offset!r}: has to be an integer from 0 to 2^64 - 1")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} on {residual.device} does not go with x "
                         f"{tuple(x.shape)} {x.dtype} on {x.device}")


def _run(x, res, args):
    """``args``: threshold, seed (signed), seed on the device or None, offset (signed)."""
    x = cuda._aligned16(x.contiguous())
    if res is not None:
        res = cuda._aligned16(res.contiguous())
    y = torch.empty_like(x)
    n = x.numel()
    if n:
        with cuda.on_device(x):
            cuda.call("slab_dropout", x, res, y, int(x.dtype == torch.bfloat16), n, *args, cuda.stream())
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, args):
        ctx.args = args
        return _run(x, residual, args)

    @staticmethod
    def backward(ctx, g):
        dx = None
        if ctx.needs_input_grad[0]:                # the mask's product again, itself differentiable where that is asked for
            dx = _Dropout.apply(g, None, ctx.args) if torch.is_grad_enabled() else _run(g, None, ctx.args)
        return dx, (g if ctx.needs_input_grad[1] else None), None


def dropout(x, p, seed, offset=0, residual=None):
    if x.dtype not in _TYPES:
        return ref.dropout(x, p, seed, offset, residual)
    if isinstance(seed, torch.Tensor):
        args = (ref.dropout_threshold(p), 0, seed.detach().clone(), _signed(offset))
    else:
        args = (ref.dropout_threshold(p), _signed(seed), None, _signed(offset))
    return _Dropout.apply(x, residual, args)
