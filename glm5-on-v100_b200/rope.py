"""Rotary cos/sin tables, with the frequency scalings of long-context models.

The table is what ``ops.rotary_embedding`` and the cache writers read: f32
``[max_position, rotary_dim]``, a row = rotary_dim/2 cosines | rotary_dim/2
sines (vLLM's ``cos_sin_cache``). Angles are formed in 64 bits: at position
180,000 an f32 angle is already off by 0.008 rad. A table is built once per
model, like a weight.
"""
from __future__ import annotations

import math

import torch


def _yarn_gain(factor: float, mscale: float) -> float:
    return 0.1 * mscale * math.log(factor) + 1.0 if factor > 1.0 else 1.0


def rope_inv_freq(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None, device=None):
    """(f64 [rotary_dim/2] frequencies, gain of cos and sin) under ``scaling``:

    None                                    base^(-2i/d)
    {"type": "linear", "factor": f}         every frequency / f
    {"type": "ntk", "factor": f}            base * f^(d/(d-2))
    {"type": "yarn", "factor": f, "original_max_position": n, "beta_fast": 32,
     "beta_slow": 1, "mscale": 1, "mscale_all_dim": 0, "attn_factor": 1}
        pairs that turn more than beta_fast times over n positions keep their
        frequency, those below beta_slow turns get it / f, a linear ramp over
        the pairs between; cos and sin times the gain
        (0.1 mscale ln f + 1) / (0.1 mscale_all_dim ln f + 1) * attn_factor.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise RuntimeError(f"rotary_dim must be even and positive (got {rotary_dim})")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64, device=device)
    kind = "none" if scaling is None else scaling.get("type")
    factor = 1.0 if scaling is None else float(scaling.get("factor", 1.0))
    if factor <= 0:
        raise RuntimeError(f"rope scaling factor must be positive (got {factor})")
    if kind == "ntk":
        if rotary_dim == 2:
            raise RuntimeError("ntk scaling needs rotary_dim > 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = torch.pow(torch.tensor(float(base), dtype=torch.float64, device=device), -2.0 * i / rotary_dim)
    if kind in ("none", "ntk"):
        return freq, 1.0
    if kind == "linear":
        return freq / factor, 1.0
    if kind != "yarn":
        raise RuntimeError(f"unknown rope scaling {kind!r}")
    n = float(scaling["original_max_position"])

    def pair_of(turns):  # the (real-valued) pair that turns this often over n positions
        return rotary_dim * math.log(n / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low = max(math.floor(pair_of(float(scaling.get("beta_fast", 32)))), 0)
    high = min(math.ceil(pair_of(float(scaling.get("beta_slow", 1)))), rotary_dim - 1)
    if high == low:
        high = low + 0.001
    slow = ((i - low) / (high - low)).clamp(0.0, 1.0)
    gain = (_yarn_gain(factor, float(scaling.get("mscale", 1))) /
            _yarn_gain(factor, float(scaling.get("mscale_all_dim", 0))) * float(scaling.get("attn_factor", 1)))
    return freq / factor * slow + freq * (1.0 - slow), gain


def rope_cos_sin_cache(rotary_dim: int, max_position: int, base: float = 10000.0, scaling: dict | None = None,
                       device=None) -> torch.Tensor:
    """f32 [max_position, rotary_dim] table (cos | sin) for ``ops.rotary_embedding``
    and the cache writers' cos_sin_cache."""
    if max_position <= 0:
        raise RuntimeError(f"max_position must be positive (got {max_position})")
    freq, gain = rope_inv_freq(rotary_dim, base, scaling, device)
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos() * gain, angle.sin() * gain], dim=1).to(torch.float32)
