"""The two ends of a language model around a stack of blocks: tokens to rows, and rows to a loss over the vocabulary without the
logits.  Not part of the reference's operators (its models look up and score with torch code outside of them).

A weight is ``[vocabulary, width]``, one for both ends or one each.  Tokens and targets are int32 or int64, on the device and read there:
one outside the vocabulary is no word.  fp32 tensors are computed in fp32 whatever ``set_fp32_compute`` says.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .ops import _check_device, _tracing

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _reduction(reduction: str) -> int:
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(_REDUCTIONS)}, got {reduction!r}")
    return _REDUCTIONS[reduction]


class EmbedTokensFunction(torch.autograd.Function):
    """The lookup as a Python Function, for ``torch.jit.trace``, which records it as one operation; any other call builds the native
    node of the same computation (csrc/host.cpp: Embed)."""

    @staticmethod
    def forward(ctx, tokens, weight, scale):
        ctx.save_for_backward(tokens)
        ctx.call = (weight.shape[0], scale)
        return _lib.host().embed_tokens(tokens, weight, scale, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        vocab, scale = ctx.call
        return None, _lib.host().embed_grad(ctx.saved_tensors[0], dy, vocab, scale), None


def embed_tokens(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[tokens]``: tokens of any shape -> ``[.., width]``, zeros for what is no word (padding, say -1).  The product is
    fp32, rounded once.  Differentiable any number of times in ``weight``; its gradient adds up a word's rows in fp32 in the tokens' order,
    which gives the same bits every time, and is zero for words without a token."""
    _check_device(weight)
    if _tracing():
        return EmbedTokensFunction.apply(tokens, weight, scale)
    return _lib.host().embed_tokens(tokens, weight, scale, True)


def embed_tokens_bwd(tokens: torch.Tensor, dy: torch.Tensor, vocab: int, scale: float = 1.0) -> torch.Tensor:
    """The gradient ``[vocab, width]`` of ``embed_tokens``'s weight from that of its result, ``dy [.., width]``."""
    _check_device(dy)
    return _lib.host().embed_grad(tokens, dy, vocab, scale)


class LinearCrossEntropyFunction(torch.autograd.Function):
    """As ``EmbedTokensFunction``, of the cross entropy (csrc/host.cpp: VocabLoss)."""

    @staticmethod
    def forward(ctx, x, weight, targets, scale, ignore_index, reduction):
        loss, lse = _lib.host().linear_cross_entropy_fwd(x, weight, targets, scale, ignore_index, reduction)
        ctx.save_for_backward(x, weight, targets, lse)
        ctx.call = (scale, ignore_index, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss):
        x, weight, targets, lse = ctx.saved_tensors
        dx, dw = _lib.host().linear_cross_entropy_bwd(x, weight, targets, lse, d_loss, *ctx.call, *ctx.needs_input_grad[:2])
        return dx, dw, None, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, scale: float = 1.0, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of the logits ``scale * x @ weight.T`` (fp32, in pieces of the vocabulary, never stored) for rows ``x [.., width]``
    and their ``targets [..]``: fp32, a value for each row (``reduction="none"``), their ``"sum"``, or the ``"mean"`` over the rows that have
    a target (0 where none has).  A row whose target is ``ignore_index`` or no word has none: its loss is 0 and its gradient is 0, whatever
    it holds, and it reaches no other; such rows are left out of the products (but up to 512 rows of 16 bits are scored where they lie).

    Differentiable once in ``x`` and ``weight``, which share one dtype.  The backward pass computes the logits again and rounds their gradient to the
    tensors' type (fp32: not at all) for the two products that read it.  fp16 keeps it relative to the largest upstream gradient of the call: what
    is below 2^-28 of that loses bits, below 2^-39 all of them, so that with ``reduction="none"`` a row whose own upstream gradient is far below
    another's has a coarser gradient than it would have alone (bf16 and fp32: not).

    Memory besides the results, for N rows of width C.  Backward: a copy of the rows (N C elements, of 6 bytes for fp32); of the logits' gradient a piece
    of the vocabulary of 1 GiB, or of 256 words where that is more; N C sums in fp32 where it is taken in several pieces; sums of a gradient for
    each part of its product's summation axis where that is split (small products; together up to 2 or 3 GiB for widths above 10000); for fp32, and
    for weights off the 16-byte grid, up to 1 GiB of weights laid out anew (256 words at least).  Forward: the same copies, and 8 bytes for each row and
    64 to 256 words of a piece, at most 2 GiB."""
    _check_device(weight)
    r = _reduction(reduction)
    if _tracing():
        return LinearCrossEntropyFunction.apply(x, weight, targets, scale, ignore_index, r)
    return _lib.host().linear_cross_entropy(x, weight, targets, scale, ignore_index, r)


def linear_cross_entropy_fwd(x, weight, targets, scale: float = 1.0, ignore_index: int = -100,
                             reduction: str = "mean") -> Tuple[torch.Tensor, torch.Tensor]:
    """``linear_cross_entropy`` with the rows' log sums: ``(loss, lse)``, lse fp32 ``[..]`` in base 2 as ``parallel_moda_fwd``'s, 0 for rows
    without a target.  As there, no graph is recorded: x and weight count as constants (a forward-mode tangent is refused)."""
    _check_device(weight)
    return _lib.host().linear_cross_entropy_fwd(x, weight, targets, scale, ignore_index, _reduction(reduction))


def linear_cross_entropy_bwd(x, weight, targets, lse, d_loss, scale: float = 1.0, ignore_index: int = -100, reduction: str = "mean",
                             need_dx: bool = True, need_dweight: bool = True) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``(dx, dweight)`` from what ``linear_cross_entropy_fwd`` was given and returned and the loss's gradient ``d_loss`` (of its shape).
    x and weight count as constants; an lse or a d_loss that requires gradients is refused, and so is any tangent."""
    _check_device(weight)
    return _lib.host().linear_cross_entropy_bwd(x, weight, targets, lse, d_loss, scale, ignore_index, _reduction(reduction), need_dx, need_dweight)
