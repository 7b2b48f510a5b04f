"""Embedding lookup with scaling and its gradient by sorted tokens (``csrc/embedding.cu``).

The gradient is summed in fp32 in the order of the positions, so it is the same bits every time.  If the table carries
``main_grad`` (a view of the flat gradient buffer set by the FSDP engine) it is written there, or added to what an earlier
micro-batch left there, which touches only the rows the batch names; otherwise autograd gets the whole gradient.

Forward mode and ``torch.func``'s transforms take the oracle; a gradient that is itself differentiated (``create_graph``) or comes
as a batch (``is_grads_batched``) is made by the library's gradient of a lookup, and always handed to autograd.
"""
from __future__ import annotations

import torch

from . import cuda

cuda.register("slab_embedding_fwd", "ppipiliifps")
cuda.register("slab_embedding_bwd", "ppipippiiiifis")
cuda._KERNELS_PER_CALL["slab_embedding_bwd"] = 3

_TYPES = (torch.float32, torch.bfloat16)
MAX_ROWS = 2 ** 30                                   # of tokens, and of the table: counted in 32 bits, in whole groups and slices


def _chunk(rows: int) -> int:
    """Sorted positions that one group of threads adds up: few where there are few, so that the SMs have work; no more than
    32, so that a frequent token's run is shared by many."""
    return 8 if rows <= 2048 else 16 if rows <= 16384 else 32


def check(tokens, weight, scale) -> float:
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"a table [vocabulary, hidden] wanted, got {tuple(weight.shape)}")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"token ids have to be int32 or int64, not {tokens.dtype}")
    if tokens.numel() > MAX_ROWS:
        raise ValueError(f"{tokens.numel()} tokens: at most 2^30 in one call")
    if tokens.device != weight.device:
        raise ValueError(f"tokens on {tokens.device}, table on {weight.device}")
    return float(scale)


def supports(weight, dtype) -> bool:
    return not cuda.transformed() and weight.dtype in _TYPES and dtype in _TYPES and weight.shape[0] <= MAX_ROWS and weight.shape[1] <= 2 ** 23


def _plain_gradient(tok, g, v: int, scale: float, dtype):
    """The table's gradient by library operations, which can be differentiated and batched."""
    inside = (tok >= 0) & (tok < v)
    g = torch.where(inside[..., None], g.float() * scale, 0.0)
    return torch.ops.aten.embedding_dense_backward(g, torch.where(inside, tok, 0), v, -1, False).to(dtype)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, dtype):
        tok = tokens.long().contiguous()
        w = weight.contiguous()
        v, h = w.shape
        out = w.new_empty((*tokens.shape, h), dtype=dtype)
        if tok.numel():
            with cuda.on_device(w):
                cuda.call("slab_embedding_fwd", tok, w, int(w.dtype == torch.bfloat16), out, int(dtype == torch.bfloat16),
                          tok.numel(), v, h, scale, cuda.status_word(w.device), cuda.stream())
        ctx.save_for_backward(tok)
        ctx.w_ref, ctx.scale, ctx.table = weight, scale, (v, h, w.dtype)
        return out

    @staticmethod
    def backward(ctx, g):
        if not ctx.needs_input_grad[1]:
            return None, None, None, None
        (tok,) = ctx.saved_tensors
        v, h, dtype = ctx.table
        if torch.is_grad_enabled() or not cuda._plain_tensor(g):
            return None, _plain_gradient(tok, g, v, ctx.scale, dtype), None, None
        rows = tok.numel()
        mg = getattr(ctx.w_ref, "main_grad", None)
        into = mg if mg is not None and mg.dtype in _TYPES and mg.is_contiguous() else None
        accumulate = into is not None and ctx.w_ref.main_grad_written
        dw = into if into is not None else g.new_empty((v, h), dtype=dtype)
        if rows == 0:
            if not accumulate:
                dw.zero_()
        else:
            g = g.contiguous()
            with cuda.on_device(g):
                chunk = _chunk(rows)
                at = (rows + 1 + (v + 31) // 32 + 3) // 4 * 4      # the sorted positions, their number, which rows; then the pieces
                scratch = g.new_empty(at + (rows + chunk - 1) // chunk * (2 * h + 2), dtype=torch.int32)
                base = scratch.data_ptr()
                cuda.call("slab_embedding_bwd", tok, g, int(g.dtype == torch.bfloat16), dw, int(dw.dtype == torch.bfloat16),
                          base, base + 4 * at, rows, chunk, v, h, ctx.scale, int(accumulate), cuda.stream())
        if into is not None:
            ctx.w_ref.main_grad_written = True
            return None, None, None, None
        return None, dw, None, None


def embedding(tokens, weight, scale: float, dtype):
    return _Embedding.apply(tokens, weight, scale, dtype)
