"""Rotary frequencies of plain and of scaled (long-context) models, for rotate_rows
and append_tokens.

The pair i of a head's first R values turns by f_i radians a position,
f_i = base^(-2 i / R). Models that were stretched to longer contexts change the
f_i, and some the size of the rotated values too; `rotary_frequencies` makes both
from the parameters that model configurations name. All arithmetic is in 64
bits, rounded to fp32 once.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

__all__ = ["rotary_frequencies"]


def _number(scaling: dict, name: str, default=None) -> float:
    v = scaling.get(name, default)
    if v is None or isinstance(v, bool) or not isinstance(v, (int, float)) or not math.isfinite(v):
        raise ValueError(f"rotary scaling needs a finite {name}")
    return float(v)


# What a scaling may hold: what the formulas below read (each kind its own), and what
# says nothing about the frequencies of a given rotary_dim and base.
_KNOWN = {"type", "rope_type", "factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor",
          "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate", "rope_theta",
          "partial_rotary_factor", "max_position_embeddings", "finetuned", "mrope_section", "mrope_interleaved"}


def _kind(scaling: Optional[dict], base: float):
    if scaling is None:
        return None
    for name in scaling:
        if name not in _KNOWN:
            raise ValueError(f"rotary scaling has {name!r}, whose effect on the frequencies is not known here")
    if scaling.get("rope_theta") is not None and _number(scaling, "rope_theta") != base:
        raise ValueError(f"rotary scaling has rope_theta {scaling['rope_theta']}, but base is {base}")
    kind = scaling.get("rope_type")
    return scaling.get("type") if kind is None else kind


def _yarn_scale(scaling: dict, factor: float) -> float:
    """The table's scale of a "yarn" scaling."""
    if scaling.get("attention_factor") is not None:
        return float(scaling["attention_factor"])

    def g(s):
        return 0.1 * s * math.log(factor) + 1 if factor > 1 else 1.0

    part, whole = (0 if scaling.get(n) is None else _number(scaling, n) for n in ("mscale", "mscale_all_dim"))
    if part and whole:
        return g(part) / g(whole)
    if (part or whole) and g(part or 1) / g(whole) != g(1):
        raise ValueError("rotary scaling takes mscale and mscale_all_dim together, or attention_factor in their place")
    return g(1)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
                       seq_len: Optional[int] = None, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq fp32 [rotary_dim / 2], attention_scale). scaling: None, or a dict whose
    "type" (or "rope_type") is

    - "linear": positions divided by "factor";
    - "dynamic": base * (factor * seq_len / n - (factor - 1)) ** (R / (R - 2)) where
      seq_len passes n = "original_max_position_embeddings";
    - "llama3": wavelengths above n / "low_freq_factor" are stretched by "factor",
      those below n / "high_freq_factor" stay, between them the two frequencies are mixed
      linearly in n / wavelength;
    - "yarn": dims that turn fewer than "beta_slow" (1) times over n positions are
      stretched by "factor", those of more than "beta_fast" (32) stay, between them mixed
      linearly in the dim, the ends moved out to whole dims unless "truncate" is False;
      attention_scale is "attention_factor", or g(1), or g(mscale) / g(mscale_all_dim) where
      both are given, with g(s) = 0.1 s ln(factor) + 1 (1 for factors up to 1). One of them
      without the other (or 0) is refused unless both readings of it, g(1) and that ratio with
      g(0) = 1 for the missing one, agree.

    Names that none of them knows are refused, and a "rope_theta" that is not `base`.
    """
    R = int(rotary_dim)
    if R <= 0 or R % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if not (math.isfinite(base) and base > 0):
        raise ValueError(f"base must be positive and finite, got {base}")
    exponent = -torch.arange(0, R, 2, dtype=torch.float64) / R
    f = torch.tensor(float(base), dtype=torch.float64) ** exponent
    m = 1.0
    kind = _kind(scaling, base)
    if kind not in (None, "default"):
        factor = _number(scaling, "factor")
        if factor <= 0:
            raise ValueError(f"factor must be positive, got {factor}")
        if kind == "linear":
            f = f / factor
        elif kind == "dynamic":
            n = _number(scaling, "original_max_position_embeddings")
            if seq_len is not None and seq_len > n and R > 2:
                stretched = float(base) * (factor * seq_len / n - (factor - 1)) ** (R / (R - 2))
                f = torch.tensor(stretched, dtype=torch.float64) ** exponent
        elif kind == "llama3":
            n = _number(scaling, "original_max_position_embeddings")
            low, high = _number(scaling, "low_freq_factor"), _number(scaling, "high_freq_factor")
            if not 0 < low < high:
                raise ValueError("low_freq_factor must be positive and below high_freq_factor")
            turns = n * f / (2 * math.pi)                       # n / wavelength
            keep = ((turns - low) / (high - low)).clamp(0, 1)
            f = f / factor * (1 - keep) + f * keep
        elif kind == "yarn":
            n = _number(scaling, "original_max_position_embeddings")
            fast, slow = _number(scaling, "beta_fast", 32), _number(scaling, "beta_slow", 1)
            if not 0 < slow < fast or base == 1:
                raise ValueError("beta_slow must be positive and below beta_fast, and base not 1")

            def dim_of(turns):          # the pair that turns so often over n positions
                return R * math.log(n / (2 * math.pi * turns)) / (2 * math.log(base))

            lo, hi = dim_of(fast), dim_of(slow)
            if scaling.get("truncate") in (None, True):
                lo, hi = math.floor(lo), math.ceil(hi)
            lo, hi = max(lo, 0), min(hi, R - 1)
            far = ((torch.arange(R // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            f = f / factor * far + f * (1 - far)
            m = _yarn_scale(scaling, factor)
        else:
            raise ValueError(f"unknown rotary scaling {kind!r}")
    return f.to(torch.float32).to(device), m
