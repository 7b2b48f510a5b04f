"""Causal attention over packed documents (``csrc/packed_attention.cu``): documents of any lengths lie one behind the other
in one buffer of rows, and a row attends to its own document only (and, with ``window``, to the last ``window`` keys of it).

:func:`pack_documents` (from offsets) or :func:`documents_from_tokens` (from token ids and an end-of-document id) makes
the plan of a batch once; every layer's forward and backward pass uses it.  The kernels' path reads nothing back to the host.

The kernels take bf16 and head widths that are multiples of 8 up to 128, with any token and head strides (slices of a
packed projection are read where they lie).  Other types and widths, and CPU tensors, take the oracle
(``reference.packed_attention``), which reads the plan back and whose scores lie in memory, 512 query rows at a time.  The
kernels have no forward mode: they refuse tangents.

Reference: the packed fine-tuning batches of ``notes/mlperf-llama/2026-04-29_llama2_70b_lora_baseline_trace_breakdown.md``.
"""
from __future__ import annotations

import math

import torch

from . import cuda

cuda.register("slab_packed_plan_words", "i")
cuda.register("slab_packed_plan", "piippp")
cuda.register("slab_packed_plan_tokens", "piilppp")
cuda.register("slab_packed_attn_fwd", "ppppppp" + "iiii" + "llllll" + "if" + "ppp")
cuda.register("slab_packed_attn_splits", "iiii")
cuda.register("slab_packed_attn_bwd", "p" * 14 + "i" + "iiii" + "llllllll" + "if" + "pp")
cuda._KERNELS_PER_CALL.update({"slab_packed_plan": 2, "slab_packed_plan_tokens": 3, "slab_packed_attn_bwd": 3})
cuda._STATUS_NAMES.update({40: "PACKED_ATTN_Q", 41: "PACKED_ATTN_KV_FULL", 42: "PACKED_ATTN_EMPTY", 43: "PACKED_ATTN_S",
                           44: "PACKED_ATTN_P", 45: "PACKED_ATTN_OUT", 46: "PACKED_ATTN_ITEM"})

TILE = 128
MAX_ROWS = 2 ** 25                                  # a row's key tiles are one item, whose end is waited for: half a second of them


class PackedDocuments:
    """The documents of one packed buffer of ``rows`` rows.  ``plan`` (CUDA): per row the first row of its document and one
    past its last, per tile of 128 rows their range, and the orders in which the kernels visit tiles; ``doc_lo`` /
    ``doc_hi`` are its first two parts.  A row of no document has an empty range, ``doc_lo = row + 1``, ``doc_hi = row``."""

    def __init__(self, rows: int, plan: torch.Tensor):
        self.rows, self.plan, self.device = rows, plan, plan.device

    @property
    def doc_lo(self) -> torch.Tensor:
        return self.plan[:self.rows]

    @property
    def doc_hi(self) -> torch.Tensor:
        return self.plan[self.rows:2 * self.rows]


def pack_documents(cu_seqlens: torch.Tensor, rows: int) -> PackedDocuments:
    """Plan of ``rows`` rows that hold documents ``s`` at ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1`` (starting at 0, not
    falling, documents may be empty; rows behind the last one belong to none).  Offsets on the GPU are checked there:
    bad ones set the status word (``cuda.check_status``) and never lead a kernel out of the buffer."""
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError("cu_seqlens has to be a one-dimensional int32 or int64 tensor of document offsets")
    if not 0 < rows <= MAX_ROWS:
        raise ValueError(f"{rows} rows: has to be 1 to {MAX_ROWS}")
    if not cu_seqlens.is_cuda:
        cu = cu_seqlens.long()
        if int(cu[0]) != 0 or int(cu[-1]) > rows or bool((cu[1:] < cu[:-1]).any()):
            raise ValueError("cu_seqlens has to start at 0, not fall and not pass the buffer's rows")
        i = torch.arange(rows)
        s = torch.searchsorted(cu[1:].contiguous(), i, right=True)
        inside = s < cu.numel() - 1
        s = s.clamp_max(max(cu.numel() - 2, 0))
        lo = torch.where(inside, cu[s], i + 1)
        hi = torch.where(inside, cu[(s + 1).clamp_max(cu.numel() - 1)], i)
        return PackedDocuments(rows, torch.cat([lo, hi]).int())
    # (offsets past 32 bits have to stay past the buffer's end)
    cu = cu_seqlens.clamp(-1, 2 ** 31 - 1) if cu_seqlens.dtype == torch.int64 else cu_seqlens
    cu = cu.to(torch.int32).contiguous()
    plan = torch.empty(cuda.lib().slab_packed_plan_words(rows), dtype=torch.int32, device=cu.device)
    with cuda.on_device(cu):
        cuda.call("slab_packed_plan", cu, cu.numel() - 1, rows, plan, cuda.status_word(cu.device), cuda.stream())
    return PackedDocuments(rows, plan)


def documents_from_tokens(tokens: torch.Tensor, end_token: int) -> PackedDocuments:
    """Plan of a batch of token rows ``[B, S]`` (int64) seen as one buffer of ``B * S`` rows: a document ends behind every
    ``end_token`` and with every row of the batch."""
    if tokens.dim() != 2 or tokens.numel() == 0 or tokens.dtype != torch.int64:
        raise ValueError("tokens has to be a non-empty [B, S] int64 tensor")
    b, s = tokens.shape
    rows = b * s
    if rows > MAX_ROWS:
        raise ValueError(f"{rows} rows: at most {MAX_ROWS}")
    tok = tokens.contiguous()
    if not tok.is_cuda:
        i = torch.arange(rows)
        start = torch.ones(rows, dtype=torch.bool)
        start[1:] = (tok.reshape(-1)[:-1] == end_token) | (i[1:] % s == 0)
        lo = torch.where(start, i, 0).cummax(0).values
        ends = torch.where(torch.cat([start[1:], torch.ones(1, dtype=torch.bool)]), i + 1, rows)
        hi = ends.flip(0).cummin(0).values.flip(0)
        return PackedDocuments(rows, torch.cat([lo, hi]).int())
    plan = torch.empty(cuda.lib().slab_packed_plan_words(rows), dtype=torch.int32, device=tok.device)
    starts = torch.empty(2 * ((rows + TILE - 1) // TILE), dtype=torch.int32, device=tok.device)
    with cuda.on_device(tok):
        cuda.call("slab_packed_plan_tokens", tok, rows, s, int(end_token), starts, plan, cuda.stream())
    return PackedDocuments(rows, plan)


def check(q, k, v, documents, scale, window) -> float:
    """Refuses what neither path computes; returns the softmax scale."""
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or v.shape != ks:
        raise ValueError(f"q [rows, heads, d], k and v [rows, groups, d] wanted, got {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}")
    rows, hq, d = qs
    if ks[0] != rows or ks[2] != d or ks[1] == 0 or hq % ks[1] or hq == 0 or d == 0:
        raise ValueError(f"q {tuple(qs)} and k {tuple(ks)} do not go together")
    if documents.rows != rows:
        raise ValueError(f"the documents' plan is for {documents.rows} rows, not {rows}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v differ in type: {q.dtype}, {k.dtype}, {v.dtype}")
    dev = documents.device
    if q.device != dev or k.device != dev or v.device != dev:
        raise ValueError("q, k, v and the documents' plan lie on different devices")
    if window < 0:
        raise ValueError(f"window {window}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"softmax scale {scale}: has to be positive and finite")
    return scale


def supports(q, k, v) -> bool:
    return q.dtype == k.dtype == v.dtype == torch.bfloat16 and q.shape[-1] % 8 == 0 and q.shape[-1] <= 128


def _readable(t):
    """``(t, token stride, head stride)``, ``t`` copied where the copy engine cannot read it as it lies: unit stride inside a
    head, other strides and the address on 16 bytes (any stride counts as such on a dimension of one)."""
    n, h, d = t.shape
    ts, hs, es = t.stride()
    if n == 1:
        ts = h * d
    if h == 1:
        hs = d
    if (es == 1 or d == 1) and ts % 8 == 0 and ts > 0 and hs % 8 == 0 and hs > 0 and t.data_ptr() % 16 == 0:
        return t, ts, hs
    return t.clone(memory_format=torch.contiguous_format), h * d, d


def forward(q, k, v, documents: PackedDocuments, scale: float, window: int = 0, grads: bool = True):
    """``(out [rows, Hq, d], rest, lse)``: ``rest`` the output's lower half (int8, most of what bf16 leaves of fp32; None without
    gradients to come), ``lse`` the base-2 log-sum-exp of the scaled scores, ``[Hq, tiles * 128]`` flat, with the kernel's
    work counter behind it."""
    rows, hq, d = q.shape
    out = q.new_empty((rows, hq, d))
    stats = hq * ((rows + TILE - 1) // TILE * TILE)
    lse = q.new_empty(stats + 1, dtype=torch.float32)
    rest = q.new_empty((rows, hq, d), dtype=torch.int8) if grads else None
    q, qt, qh = _readable(q)
    k, kt, kh = _readable(k)
    v, vt, vh = _readable(v)
    with cuda.on_device(q):
        cuda.call("slab_packed_attn_fwd", q, k, v, out, rest, lse, documents.plan, rows, hq, k.shape[1], d, qt, qh, kt, kh, vt, vh,
                  min(window, rows), scale, lse.data_ptr() + 4 * stats, cuda.status_word(q.device), cuda.stream())
    return out, rest, lse


def backward(q, k, v, out, rest, lse, dout, documents: PackedDocuments, scale: float, window: int = 0):
    """``(dq, dk, dv)`` from what the forward pass took and returned.  Where a group's heads are cut into parts
    (long documents, few key tiles for the SMs), the parts' sums are kept in fp32 and added up in their order."""
    rows, hq, d = q.shape
    hkv = k.shape[1]
    dq = q.new_empty((rows, hq, d))
    dk = q.new_empty((rows, hkv, d))
    dv = torch.empty_like(dk)
    stats = lse.numel() - 1
    delta = q.new_empty(stats + 3, dtype=torch.float32)         # and two work counters, the number of parts
    q, qt, qh = _readable(q)
    k, kt, kh = _readable(k)
    v, vt, vh = _readable(v)
    dout, gt, gh = _readable(dout)
    with cuda.on_device(q):
        splits = cuda.lib().slab_packed_attn_splits(rows, hq, hkv, min(window, rows))
        partial = q.new_empty(splits * 2 * dk.numel(), dtype=torch.float32) if splits > 1 else None
        cuda.call("slab_packed_attn_bwd", q, k, v, out, rest, dout, lse, documents.plan, dq, dk, dv, delta,
                  delta.data_ptr() + 4 * stats, partial, splits, rows, hq, hkv, d, qt, qh, kt, kh, vt, vh, gt, gh,
                  min(window, rows), scale, cuda.status_word(q.device), cuda.stream())
        if splits > 1:
            cuda.LAUNCHES[0] += 1
    return dq, dk, dv


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, documents, scale, window):
        q, k, v = (_readable(t)[0] for t in (q, k, v))         # copied once, if at all, for both passes
        out, rest, lse = forward(q, k, v, documents, scale, window)
        ctx.save_for_backward(q, k, v, out, rest, lse)
        ctx.documents, ctx.scale, ctx.window = documents, scale, window
        return out

    @staticmethod
    @cuda.first_order
    def backward(ctx, g):
        return backward(*ctx.saved_tensors, g, ctx.documents, ctx.scale, ctx.window) + (None, None, None)


def attention(q, k, v, documents: PackedDocuments, scale: float, window: int = 0):
    # (there is no forward mode: tangents go to the Function, which refuses them)
    if not (cuda.forward_mode() or torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return forward(q, k, v, documents, scale, window, grads=False)[0]
    return _PackedAttention.apply(q, k, v, documents, scale, window)
