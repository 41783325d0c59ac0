"""Rotary positions of queries and keys: not part of the reference's operators (its models rotate with torch code outside
of them), here one launch for both tensors, forward and backward.

A head's first ``dim`` elements turn in pairs by ``2 pi * position * rate``; the product and its fraction are taken in 64
bits, so that a position of a million is as exact as the first.  ``Rotary`` holds the rates (turns per position), which also
carry what stretches a model to longer contexts.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import _check_device, _tracing


class Rotary:
    """What the rotation of a model is: ``dim`` elements of each head, in pairs ``(2i, 2i + 1)`` with ``interleaved``, else
    ``(i, i + dim / 2)``, pair ``i`` at ``base ** (-2 i / dim) / (2 pi)`` turns per position.

    ``scaling`` by ``factor``, for contexts longer than the ``original_length`` that a model was trained on:
      * ``"linear"``: every rate divided by the factor;
      * ``"ntk"``: the base times ``factor ** (dim / (dim - 2))``, which divides the slowest rate by the factor and leaves
        the fastest;
      * ``"by_parts"``: pairs that make fewer than ``slow`` turns over the original length are divided by the factor, those with more
        than ``fast`` stay, in between a blend linear in the turns; the rotated elements are multiplied by ``0.1 ln(factor) + 1``.
    ``amplitude`` (on the rotated elements) and ``rates`` replace what the rules above give.

    The rates stay on the host in 64 bits; each device gets a copy at its first call (before a graph capture make one
    ordinary call, as for every operator of this package; a captured call reads that copy at every replay: keep the ``Rotary`` as long
    as the graph).  A ``Rotary`` may be dropped while calls on any stream are still under way."""

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, scaling: Optional[str] = None, factor: float = 1.0,
                 original_length: Optional[int] = None, slow: float = 1.0, fast: float = 32.0, amplitude: Optional[float] = None,
                 rates: Optional[Sequence[float]] = None):
        if dim <= 0 or dim % 2:
            raise ValueError(f"dim must be positive and even, got {dim}")
        if scaling not in (None, "linear", "ntk", "by_parts"):
            raise ValueError(f"unknown scaling {scaling!r}")
        if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
            raise ValueError(f"base and factor must be positive, got {base} and {factor}")
        if scaling == "ntk" and dim == 2:
            raise ValueError("a single pair has no slower one: scale it linearly")
        if scaling == "by_parts" and (not original_length or original_length <= 0 or not slow < fast):
            raise ValueError("scaling by parts needs the original length, and slow < fast")
        self.dim, self.interleaved = int(dim), bool(interleaved)
        self.amplitude = 1.0
        if rates is not None:
            table = torch.as_tensor(rates, dtype=torch.float64).reshape(-1).cpu().clone()
            if table.numel() * 2 != dim or not bool(torch.isfinite(table).all()):
                raise ValueError(f"rates must be {dim // 2} finite values")
        else:
            if scaling == "ntk":
                base = base * factor ** (dim / (dim - 2))
            table = torch.tensor([base ** (-2 * i / dim) / (2 * math.pi) for i in range(dim // 2)], dtype=torch.float64)
            if scaling == "linear":
                table = table / factor
            elif scaling == "by_parts":
                keep = ((table * original_length - slow) / (fast - slow)).clamp(0, 1)
                table = table / factor * (1 - keep) + table * keep
                self.amplitude = 0.1 * math.log(factor) + 1.0
        if amplitude is not None:
            self.amplitude = float(amplitude)
        self._host = table
        self._on: dict = {}

    def rates(self, device) -> torch.Tensor:
        """The ``dim / 2`` rates in 64 bits on ``device``."""
        t = self._on.get(device)
        if t is None:
            with torch.inference_mode(False):  # a tensor made in inference mode could not be saved for a backward pass later
                t = self._on[device] = self._host.to(device)
        return t

    def __getstate__(self):
        return {**self.__dict__, "_on": {}}

    def __repr__(self):
        return f"Rotary(dim={self.dim}, interleaved={self.interleaved}, amplitude={self.amplitude})"


class RotaryFunction(torch.autograd.Function):
    """The rotation as a Python Function, for ``torch.jit.trace``, which records it as one operation; any other call builds the
    native node of the same computation (csrc/host.cpp: Rotate)."""

    @staticmethod
    def forward(ctx, q, k, rotary, positions, moda_group_num, inverse):
        ctx.call = (rotary, moda_group_num, inverse)
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        x = q if q is not None else k
        return _lib.host().apply_rotary(q, k, rotary.rates(x.device), rotary.dim, rotary.amplitude, rotary.interleaved, positions,
                                        moda_group_num, inverse, False)

    @staticmethod
    def backward(ctx, dq, dk):
        if dq is None and dk is None:
            return (None,) * 6
        rotary, G, inverse = ctx.call
        return (*RotaryFunction.apply(dq, dk, rotary, ctx.saved_tensors[0], G, not inverse), None, None, None, None)


def apply_rotary(q: Optional[torch.Tensor], k: Optional[torch.Tensor], rotary: Rotary, positions: Optional[torch.Tensor] = None,
                 moda_group_num: int = 1, inverse: bool = False) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """``q [B, T*moda_group_num, Hq, D]`` and ``k [B, T, H, D]`` (either may be None) rotated by their tokens' positions: int32 or
    int64 ``[T]`` or ``[B, T]``, by default ``0 .. T - 1``; of a packed batch pass the positions within each sequence.  Row ``r`` of
    ``q`` belongs to token ``r // moda_group_num``, as in ``parallel_moda``; for ``parallel_attn``'s ``[B, T, HQ, D]`` leave it at 1.
    ``inverse`` turns back (with an amplitude other than 1: not the inverse, but the gradient).  Returns ``(q', k')``, new
    tensors, differentiable any number of times.  Any strides are read in place."""
    x = q if q is not None else k
    if x is None:
        raise ValueError("q, k or both")
    _check_device(x)
    if _tracing():
        return RotaryFunction.apply(q, k, rotary, positions, moda_group_num, inverse)
    return _lib.host().apply_rotary(q, k, rotary.rates(x.device), rotary.dim, rotary.amplitude, rotary.interleaved, positions,
                                    moda_group_num, inverse, True)
