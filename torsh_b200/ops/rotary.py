"""Rotary positions with explicit positions: both pairings, part of the head, and frequencies scaled for long contexts.

Kernel: ``csrc/kernels/rotary.cu`` (queries and keys in one launch, forward and backward); CPU tensors run the same formula in
PyTorch. :func:`~torsh_b200.ops.elementwise.rope` is the fixed form for training (adjacent pairs of whole heads, positions
``0 .. S-1``); this one takes the position of every token, as decoding, packed batches and trees of drafted tokens need, and works
angles out in 64 bits, so that position 1 000 000 is as exact as position 1. The reference's rotary layer and its position
interpolation: ``crates/torsh-nn/src/layers/embedding.rs:372-430``.
"""
from __future__ import annotations

import math

import torch

from .. import _native as nv

SCALINGS = ("none", "linear", "ntk", "yarn", "wavelength")


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, trained_len: int = 4096,
                       low: float = 1.0, high: float | None = None, device=None) -> tuple[torch.Tensor, float]:
    """``(freqs, magnitude)`` for :func:`rotary`: radians per position of each of the ``dim // 2`` pairs in float64, and the factor
    on the turned columns.

    A model trained on ``trained_len`` positions reaches ``factor`` times as far with

    * ``"linear"``      every frequency divided by ``factor`` (position interpolation)
    * ``"ntk"``         the base raised to ``base * factor^(dim / (dim - 2))``: fast pairs keep their rate, the slowest is divided by ``factor``
    * ``"yarn"``        pairs that turn more than ``high`` (32) times over the trained length keep their rate, those below ``low`` (1) are
      divided by ``factor``, a linear ramp over the pair index between; ``magnitude = 0.1 ln(factor) + 1``
    * ``"wavelength"``  the same two ends (``high`` 4), the ramp linear in the number of turns
    """
    if dim < 0 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim must be even, got {dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (factor >= 1.0 and base > 1.0 and trained_len > 0):
        raise ValueError("rotary_frequencies: factor >= 1, base > 1 and trained_len > 0")
    magnitude = 1.0
    if scaling == "ntk":
        base = base * factor ** (dim / max(dim - 2, 1))
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    freqs = base ** (-i / max(dim, 1))
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        high = 32.0 if high is None else high
        at = lambda turns: dim * math.log(trained_len / (turns * 2 * math.pi)) / (2 * math.log(base))   # noqa: E731  pair that turns so often
        first, last = max(math.floor(at(high)), 0), min(math.ceil(at(low)), dim - 1)
        ramp = ((i / 2 - first) / max(last - first, 0.001)).clamp(0, 1)
        freqs = freqs / factor * ramp + freqs * (1 - ramp)
        magnitude = 0.1 * math.log(factor) + 1.0
    elif scaling == "wavelength":
        high = 4.0 if high is None else high
        if not high > low:
            raise ValueError("rotary_frequencies: high must be above low")
        keep = ((trained_len * freqs / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        freqs = freqs / factor * (1 - keep) + freqs * keep
    return freqs.to(device), magnitude


def _rotary_plain(x, positions, freqs, interleaved, magnitude, inverse):
    """The formula in fp32 with angles in fp64; the CPU path and the test oracle."""
    rot = 2 * freqs.numel()
    angle = positions.double()[..., None, None] * freqs
    dt = torch.float64 if x.dtype == torch.float64 else torch.float32
    cos, sin = (angle.cos() * magnitude).to(dt), (angle.sin() * (-magnitude if inverse else magnitude)).to(dt)
    xf = x.to(dt)
    r, rest = xf[..., :rot], xf[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, w], -1).reshape(r.shape) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, rest], -1).to(x.dtype)


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool = True,
           magnitude: float = 1.0):
    """Turns queries and keys by their positions; returns ``(q', k')`` (``k'`` is None where ``k`` is).

    ``q`` is ``[..., Hq, D]``, ``k`` ``[..., Hk, D]`` with the same leading dimensions (``[B, T]`` or ``[tokens]``), ``positions``
    integers of those dimensions or fewer (``[T]`` serves every sequence). ``freqs`` (:func:`rotary_frequencies`) has one entry per
    pair: ``2 * len(freqs)`` columns of ``D`` turn, the rest pass through. ``interleaved`` pairs columns ``(2i, 2i + 1)``, as
    :func:`~torsh_b200.ops.elementwise.rope` does; otherwise ``(i, i + len(freqs))``. Differentiable in ``q`` and ``k``; forward-mode derivatives, and calls whose
    ``freqs`` require a gradient, are computed in PyTorch.
    """
    if q.is_cuda:
        out = (nv._decode or nv.decode_calls()).rotary(q, k, positions, freqs, interleaved, magnitude)
        if out is not None:
            return out
    # not as the kernel takes it: refused, converted, or computed here
    shape = q.shape
    if len(shape) < 2 or (k is not None and (k.shape[:-2] != shape[:-2] or k.shape[-1] != shape[-1] or k.dtype != q.dtype)):
        raise ValueError("rotary: q and k are [..., heads, D] of one type with the same leading dimensions and D")
    if freqs.dim() != 1 or 2 * freqs.numel() > shape[-1]:
        raise ValueError(f"rotary: freqs has one entry for each pair of at most {shape[-1]} columns")
    if positions.dtype is not torch.int64 and (positions.is_floating_point() or positions.dtype == torch.bool):
        raise TypeError("rotary: positions are integers")
    lead = shape[:-2]
    if positions.shape != lead:
        try:
            positions = positions.expand(lead)
        except RuntimeError:
            raise ValueError(f"rotary: positions {tuple(positions.shape)} do not fit {tuple(lead)}") from None
    at = q.get_device()
    if positions.get_device() != at or freqs.get_device() != at or (k is not None and k.get_device() != at):
        raise ValueError("rotary: all tensors are on one device")
    if q.is_cuda:
        with torch.cuda.device(q.device):
            out = nv.decode_calls().rotary(q, k, positions.to(torch.int64).contiguous(), freqs.to(torch.float64).contiguous(), interleaved, magnitude)
        if out is not None:
            return out
    f = freqs.to(torch.float64)
    return tuple(None if x is None else _rotary_plain(x, positions, f, interleaved, magnitude, False) for x in (q, k))
