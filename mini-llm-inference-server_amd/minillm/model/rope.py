"""Rotary-embedding frequencies, plain and scaled for long contexts, and the rotation itself in torch operations
(reference src/minillm/model/rope.py:16-42 has the plain and the llama3 frequencies).

inv_freq[i] = theta^(-2i / R) for the R rotated dims of a head.  Scaling by `factor` s (rope_type):
  linear  every frequency divided by s (positions interpolated);
  llama3  wavelengths 2*pi / inv_freq longer than original_len / low_freq_factor are divided by s, those shorter than
          original_len / high_freq_factor are kept, and the band between is a linear blend in original_len / wavelength;
  yarn    pairs that turn more than beta_fast times over the original length are kept, those that turn less than beta_slow
          times are divided by s, with a linear blend over the pair's index between; cosines and sines are scaled by
          0.1 ln(s) + 1 (or attention_factor; mscale and mscale_all_dim give the ratio of 0.1 m ln(s) + 1).
"""

from __future__ import annotations

import math

import torch


def compute_inv_freq(config) -> torch.Tensor:
    dim = config.rotary_dim
    exponents = torch.arange(0, dim, 2, dtype=torch.int64, device="cpu").float() / dim
    inv_freq = 1.0 / (config.rope_theta ** exponents)
    sc = config.rope_scaling
    if sc is None:
        return inv_freq
    kind = sc["rope_type"]
    if kind == "linear":
        return inv_freq / sc["factor"]
    if kind == "yarn":
        return _yarn(config, inv_freq)
    if kind != "llama3":
        raise NotImplementedError(f"rope_type {kind!r}")
    factor, lo, hi = sc["factor"], sc["low_freq_factor"], sc["high_freq_factor"]
    orig = sc["original_max_position_embeddings"]
    wavelen = 2 * math.pi / inv_freq
    long_wave = wavelen > orig / lo
    short_wave = wavelen < orig / hi
    blend = (orig / wavelen - lo) / (hi - lo)
    mid = (1 - blend) * inv_freq / factor + blend * inv_freq
    out = torch.where(long_wave, inv_freq / factor, mid)
    return torch.where(short_wave, inv_freq, out)


def _yarn(config, inv_freq: torch.Tensor) -> torch.Tensor:
    sc, dim = config.rope_scaling, config.rotary_dim
    orig = sc.get("original_max_position_embeddings") or config.max_position_embeddings

    def pair_that_turns(times: float) -> float:
        """The (fractional) pair that turns so many times over the original length."""
        return dim * math.log(orig / (times * 2 * math.pi)) / (2 * math.log(config.rope_theta))

    low = pair_that_turns(sc.get("beta_fast") or 32.0)
    high = pair_that_turns(sc.get("beta_slow") or 1.0)
    if sc.get("truncate", True):
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    high = high + 0.001 if high == low else high
    slow = ((torch.arange(dim // 2, dtype=torch.float32) - low) / (high - low)).clamp(0, 1)
    return inv_freq / sc["factor"] * slow + inv_freq * (1 - slow)


def attention_factor(config) -> float:
    """What cosines and sines are scaled by: 1 but for yarn."""
    sc = config.rope_scaling
    if sc is None or sc["rope_type"] != "yarn":
        return 1.0
    if sc.get("attention_factor") is not None:
        return float(sc["attention_factor"])

    def scale(m: float) -> float:
        return 0.1 * m * math.log(sc["factor"]) + 1.0 if sc["factor"] > 1 else 1.0

    if sc.get("mscale") and sc.get("mscale_all_dim"):
        return scale(sc["mscale"]) / scale(sc["mscale_all_dim"])
    return scale(1.0)


def rotate(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool, factor: float) -> torch.Tensor:
    """`kernels.rotary` of one tensor x [B, heads, T, Dh] in torch operations, for other devices and types and for gradients:
    angles in 64 bits, the rotation in float32 (float64 of float64), one rounding."""
    ang = positions[:, None, :, None].double() * inv_freq.double()
    wide = torch.promote_types(x.dtype, torch.float32)
    cos, sin = ((f(ang) * factor).to(wide) for f in (torch.cos, torch.sin))
    rot = 2 * inv_freq.shape[0]
    y = x[..., :rot].to(wide)
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
    else:
        a, b = y.chunk(2, dim=-1)
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([y.to(x.dtype), x[..., rot:]], dim=-1)
