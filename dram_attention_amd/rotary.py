"""Rotary positions of queries and keys on the HIP kernel: interleaved and half layouts, a part of each head, frequencies
scaled for long contexts, with gradients.

Beside ``llama.apply_rope``, which turns whole heads of one sequence by rows of a table (the rotation of the reference's
model, evaluation/dram-attention/model.py:81-136): here angles are formed in the kernel from positions and
frequencies, in 64 bits, so there is no table and a position may be any.
"""

from __future__ import annotations

import math

import torch

from . import _lib

LAYOUTS = {"interleaved": 0, "half": 1}


def rotary_frequencies(rotary_dim: int, theta: float = 500000.0, scaling: dict | None = None,
                       device="cuda") -> tuple[torch.Tensor, float]:
    """(freqs, factor) for :func:`rotate`: radians per position of each of the rotary_dim / 2 pairs, float64, and the
    factor on cosine and sine.

    ``scaling``: None, or a dict with ``"type"`` and

      "linear"  ``factor``: all frequencies slowed alike
      "ntk"     ``factor``: the base raised so that the slowest pair is slowed by the factor and the fastest not at all
      "llama3"  ``factor`` (8), ``original_length`` (8192), ``low_freq_factor`` (1), ``high_freq_factor`` (4): wavelengths
                above original_length / low slowed, below original_length / high kept, a linear blend between
                (evaluation/dram-attention/model.py:81-105)
      "yarn"    ``factor``, ``original_length``, ``beta_fast`` (32), ``beta_slow`` (1), ``attention_factor`` (0.1 ln factor
                + 1): pairs that turn more than beta_fast times within original_length kept, fewer than beta_slow times
                slowed, a ramp over the pairs between
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"channels turn in pairs (got rotary_dim {rotary_dim})")
    if not (math.isfinite(theta) and theta > 1):
        raise ValueError(f"theta must be above 1 (got {theta})")
    scaling = dict(scaling or {"type": None})
    kind = scaling.pop("type", None)
    base, factor = float(theta), 1.0
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)

    def take(name, default=None):
        value = scaling.pop(name, default)
        if value is None or not value > 0:
            raise ValueError(f"scaling {kind!r} needs a {name} above 0 (got {value})")
        return float(value)

    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("scaling 'ntk' needs two pairs")
        base *= take("factor") ** (rotary_dim / (rotary_dim - 2))
    freqs = base ** (-2.0 * pair / max(rotary_dim, 1))
    if kind == "linear":
        freqs = freqs / take("factor")
    elif kind == "llama3":
        by, length = take("factor", 8.0), take("original_length", 8192.0)
        low, high = take("low_freq_factor", 1.0), take("high_freq_factor", 4.0)
        if not high > low:
            raise ValueError("scaling 'llama3' needs high_freq_factor above low_freq_factor")
        kept = ((length * freqs / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        freqs = (1 - kept) * freqs / by + kept * freqs
    elif kind == "yarn":
        by, length = take("factor"), take("original_length")
        fast, slow = take("beta_fast", 32.0), take("beta_slow", 1.0)
        given = scaling.pop("attention_factor", None)
        factor = float(given) if given is not None else 0.1 * math.log(by) + 1.0 if by > 1 else 1.0

        def pair_that_turns(n):     # n times within the original length
            return rotary_dim * math.log(length / (n * 2 * math.pi)) / (2 * math.log(theta))

        first = max(math.floor(pair_that_turns(fast)), 0)
        last = min(math.ceil(pair_that_turns(slow)), rotary_dim - 1)
        slowed = ((pair - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        freqs = (1 - slowed) * freqs + slowed * freqs / by
    elif kind not in (None, "ntk"):
        raise ValueError(f"unknown scaling {kind!r}")
    if scaling:
        raise ValueError(f"scaling {kind!r} does not take {', '.join(scaling)}")
    return freqs.to(device), factor


def layout_code(layout: str) -> int:
    try:
        return LAYOUTS[layout]
    except (KeyError, TypeError):
        raise ValueError(f"layout must be 'interleaved' or 'half' (got {layout!r})") from None


def rotate(xq: torch.Tensor, xk: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, *,
           layout: str = "interleaved", factor: float = 1.0):
    """(xq, xk) with the first 2 * len(freqs) channels of every head turned by their token's position; the others are
    copied.  Differentiable in xq and xk.

    xq (tokens, heads, head_dim) or (batch, tokens, heads, head_dim), xk likewise with heads of its own, or None;
    positions int32 or int64, one per token: (tokens,), or (batch, tokens).  ``layout``: which channels turn together,
    2i and 2i + 1 ("interleaved", as llama.py's checkpoints have them) or i and i + len(freqs) ("half").  ``freqs`` and
    ``factor`` are :func:`rotary_frequencies`'s.  bf16, fp16 or fp32 with any strides; products in fp32, rounded once.
    A call with gradients that is captured into a graph refuses leaves that an eager graph still holds.
    """
    return _lib.host().rotate(xq, xk, positions, freqs, layout_code(layout), float(factor), 0)


def rotate_(xq: torch.Tensor, xk: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, *,
            layout: str = "interleaved", factor: float = 1.0):
    """:func:`rotate` in place, without gradients; returns (xq, xk)."""
    _lib.host().rotate(xq, xk, positions, freqs, layout_code(layout), float(factor), 1)
    return xq, xk
