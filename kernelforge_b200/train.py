"""Training operators around an MoE layer's expert products, in bf16, fp16 or fp32.

The layer's ``kernel(...)`` routes, sorts, multiplies and combines in one call on FP8
weights, without gradients.  These operators are its parts around a caller's own expert
products (for instance a grouped matrix product over the sorted rows), with their
gradients, and the rows and activations that the backward pass needs kept in 8 bits:

    idx, weight = train.route(logits, bias, 2.5)                 # differentiable in the logits
    rows, order = train.sort_tokens(x, idx, 256, row_align=16)   # differentiable in x
    act = train.swiglu(rows_times_w13)                           # keeps its input in 8 bits
    out = train.combine_tokens(act_times_w2, order, weight)      # differentiable in rows and weights

A product written as its own autograd function can keep its operands in 8 bits as well:
``pack8`` keeps the token rows once, and ``restore8(kept, order)`` gives them back in expert
order; ``swiglu_backward8`` returns the activation along with the gradient.

Every call runs on the current stream of its tensors' device, allocates its outputs and
scratch from torch's caching allocator and never synchronises (but to read a
``routed_scaling_factor`` that is a CUDA tensor; pass a number), so it can be captured into
a CUDA graph, after one call outside a capture (the library's set-up on a device).  A
captured call on a leaf tensor that an eager autograd graph of the default stream still holds
raises, as its backward pass could not be captured (a graph made on a side stream does no harm;
arguments computed from such a leaf, a cast or a view of it, are not looked through).  Errors raise
``RuntimeError``.  Sums are fp32 in a fixed order: equal inputs give equal bits.  The gradients
are not differentiable again: a backward pass with ``create_graph=True`` raises.  There are no
forward-mode derivatives: a tensor that carries a tangent (``torch.autograd.forward_ad``) raises, but
in ``pack8`` and ``swiglu_pack8``, which pass no derivative at all.

The reference has no training path; its routing, sort and combine are inside ``kernel``
(``solution/triton/kernel.py:1842-1925``).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import binding as B

BLOCK = 128   # columns of a row that share an exponent in 8 bits


class TokenOrder(NamedTuple):
    """Where ``sort_tokens`` put each (token, choice) pair; all int32 on the tokens' device.

    The operators take it as ``sort_tokens`` gave it.  In an order put together otherwise, rows and
    pairs out of range count as none; rows that ``row_pair`` and ``pair_row`` disagree about are undefined.
    """
    pair_row: torch.Tensor   # [T, K] row of each pair, -1 without one
    row_pair: torch.Tensor   # [R] pair t * K + k of each row, -1 without one
    counts: torch.Tensor     # [E] pairs of each local expert
    starts: torch.Tensor     # [E + 1] first row of each expert's segment, and their end


class Rows8(NamedTuple):
    """Rows in 8 bits: ``codes * 2 ** (exponents - 127)``, one exponent per row and 128 columns.

    ``pack8`` counts the columns from the row's first, ``swiglu_pack8`` from the first of each half; the shapes
    alone do not tell the two apart, so each returns a type of its own, and an operator that reads the other
    layout refuses it (unless a half is a multiple of 128 wide, where both are the same).  A ``Rows8`` that a
    caller puts together from its parts is read as the operator reads rows.
    """
    codes: torch.Tensor      # e4m3 [R, W]
    exponents: torch.Tensor  # uint8 [R, ceil(W / 128)] (for SwiGLU's input 2 ceil(I / 128): up's, then gate's)
    dtype: torch.dtype       # of the rows they were made from


class WholeRows8(Rows8):
    """What ``pack8`` returns: blocks begin at the row's first column."""
    __slots__ = ()


class HalvesRows8(Rows8):
    """What ``swiglu_pack8`` returns: blocks begin at the first column of each half."""
    __slots__ = ()


def _refuse_layout(kept: Rows8, other: type, what: str) -> None:
    if isinstance(kept, other) and kept.codes.shape[-1] % (2 * BLOCK):
        raise RuntimeError(f"{what} reads rows whose blocks of {BLOCK} columns begin elsewhere than those of this "
                           f"{type(kept).__name__} of {kept.codes.shape[-1]} columns")


def _factor(v) -> float:
    if isinstance(v, torch.Tensor) and v.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a routed_scaling_factor that is a CUDA tensor has to be read back, which a stream capture "
                           "does not allow: pass a number")
    return B._scalar_float(v)


def route(routing_logits: torch.Tensor, routing_bias: torch.Tensor, routed_scaling_factor):
    """As ``binding.route``, with weights that are differentiable in the logits.

    The choice of experts has no gradient, and the bias takes part in the choice only.
    """
    return B.extension().route(routing_logits, routing_bias, _factor(routed_scaling_factor))


def route_backward(routing_logits: torch.Tensor, topk_idx: torch.Tensor, grad_weight: torch.Tensor,
                   routed_scaling_factor) -> torch.Tensor:
    """f32 ``[T, 256]``: the gradient of the routing weights (f32 ``[T, 8]``) in the logits.

    Ids outside [0, 256) count as no choice.
    """
    return B.extension().route_backward(routing_logits, topk_idx, grad_weight, _factor(routed_scaling_factor))


def sort_tokens(x: torch.Tensor, topk_idx: torch.Tensor, num_experts: int, expert_offset: int = 0, *,
                row_align: int = 1, max_rows: Optional[int] = None):
    """The tokens' rows in expert order: ``(rows [R, H], TokenOrder)``; differentiable in ``x``.

    ``x`` ``[T, H]``, ``topk_idx`` int32 ``[T, K]`` with global expert ids, K from 1 to 16.  The local
    experts are ``[expert_offset, expert_offset + num_experts)`` within the layer's 256; a pair with
    any other id (such as -1 for a masked token) gets no row.  Each expert's rows are in (token,
    choice) order and start at a multiple of ``row_align`` (1 to 1024); rows that belong to no pair are zero.

    ``R`` is what the worst routing needs, ``T * K + min(T * K, num_experts) * (row_align - 1)`` cut to a
    multiple of ``row_align``, or ``max_rows`` (a multiple of it): then pairs whose row would lie past
    the end are dropped.  ``order.counts`` counts them still, so drops are visible.  An id that a
    token repeats is a pair of its own.
    """
    rows, pair_row, row_pair, counts, starts = B.extension().sort_tokens(
        x, topk_idx, num_experts, expert_offset, row_align, max_rows)
    return rows, TokenOrder(pair_row, row_pair, counts, starts)


def sort_tokens_backward(grad_rows: torch.Tensor, order: TokenOrder) -> torch.Tensor:
    """``[T, H]``: the gradient of ``sort_tokens`` in ``x`` (the sum of each token's rows)."""
    return B.extension().sort_tokens_backward(grad_rows, order.pair_row, order.row_pair)


def combine_tokens(rows: torch.Tensor, order: TokenOrder, topk_weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_k topk_weight[t, k] * rows[order.pair_row[t, k]]``; differentiable in rows and weights.

    ``topk_weight`` f32 ``[T, K]``, or None for weights of 1.  Pairs without a row contribute nothing
    (a token without any gives zeros), and rows without a pair are not read: they may hold anything.
    """
    return B.extension().combine_tokens(rows, order.pair_row, order.row_pair, topk_weight)


def combine_tokens_backward(grad_output: torch.Tensor, rows: torch.Tensor, order: TokenOrder,
                            topk_weight: torch.Tensor):
    """``(grad_rows [R, H], grad_weight f32 [T, K])`` of ``combine_tokens``; rows without a pair get zeros."""
    return B.extension().combine_tokens_backward(grad_output, rows, order.pair_row, order.row_pair, topk_weight)


def pack8(x: torch.Tensor) -> Rows8:
    """Rows ``[R, W]`` in 8 bits, a value's error at most 2^-4 of it (2^-10 of the block's scale near zero).

    Values that are not finite are kept as NaN; the others of their block keep their precision.
    No gradient passes.
    """
    codes, exponents = B.extension().pack8(x)
    return WholeRows8(codes, exponents, x.dtype)


def restore8(kept: Rows8, order: Optional[TokenOrder] = None) -> torch.Tensor:
    """The rows that ``kept`` (of ``pack8``) stands for, or with ``order`` its tokens' rows in expert order (zeros elsewhere)."""
    _refuse_layout(kept, HalvesRows8, "restore8")
    return B.extension().restore8(kept.codes, kept.exponents, kept.dtype, order.pair_row if order is not None else None,
                                  order.row_pair if order is not None else None)


def swiglu(h: torch.Tensor) -> torch.Tensor:
    """``up * silu(gate)`` of ``h`` ``[R, 2 I]`` = [up | gate]; the backward pass reads ``h`` from 8 bits.

    So its gradient is that of the kept values, in fp32 too: for normally distributed ``h`` it differs from the
    gradient at ``h`` by 3 % (root mean square; cosine 0.9995).  For that one, take SwiGLU from torch's own
    operations.  A sigmoid below 2^-126 (a gate under -87) may count as zero.
    """
    return B.extension().swiglu(h)


def swiglu_pack8(h: torch.Tensor):
    """``(act [R, I], Rows8)``: SwiGLU and its input in 8 bits, in one pass.  No gradient passes."""
    act, codes, exponents = B.extension().swiglu_pack8(h)
    return act, HalvesRows8(codes, exponents, h.dtype)


def swiglu_backward8(kept: Rows8, grad_act: torch.Tensor, need_act: bool = True):
    """``(grad_h [R, 2 I], act [R, I] or None)`` from SwiGLU's kept input, in the type of ``grad_act``."""
    _refuse_layout(kept, WholeRows8, "swiglu_backward8")
    return tuple(B.extension().swiglu_backward8(kept.codes, kept.exponents, grad_act, need_act))
