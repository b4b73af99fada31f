"""RoPE angle tables in vLLM's `cos_sin_cache` layout ([max_pos, d]: cos | sin by halves).

In serving the table comes from the model's own rotary module (vllm_ttkv/impl.py:326-352 in the
reference); this builder exists for benchmarks and tests, with the public Llama 3 rope-scaling
rule (Llama-3.2-3B: theta 500000, factor 32, low/high frequency factors 1 and 4, original
context 8192).

`Rotary` is what the rotations without a table take (`kernels.rotary_scaled`,
`kernels.octet_write_paged`): frequencies in revolutions per position, in 64 bits, so that the angles
of far positions stay exact; `scaled_rotary` makes one by the usual rules for long contexts.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

LLAMA32_3B_ROPE = dict(theta=500000.0, factor=32.0, low_freq_factor=1.0, high_freq_factor=4.0,
                       original_max_position=8192)


def llama3_inv_freq(d: int = 128, theta: float = 500000.0, factor: float = 32.0,
                    low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                    original_max_position: int = 8192) -> torch.Tensor:
    inv = 1.0 / (theta ** (torch.arange(0, d, 2, dtype=torch.float32) / d))
    wavelen = 2 * math.pi / inv
    smooth = (original_max_position / wavelen - low_freq_factor) / (high_freq_factor
                                                                    - low_freq_factor)
    mid = (1 - smooth) * inv / factor + smooth * inv
    lo_wl = original_max_position / low_freq_factor
    hi_wl = original_max_position / high_freq_factor
    return torch.where(wavelen < hi_wl, inv, torch.where(wavelen > lo_wl, inv / factor, mid))


def cos_sin_cache(max_pos: int, d: int = 128, inv_freq: torch.Tensor | None = None,
                  device="cpu") -> torch.Tensor:
    """[max_pos, d] fp32: cos(t * inv_freq) in columns [0, d/2), sin in [d/2, d)."""
    inv = llama3_inv_freq(d, **LLAMA32_3B_ROPE) if inv_freq is None else inv_freq
    t = torch.arange(max_pos, dtype=torch.float32)
    f = torch.outer(t, inv.to(torch.float32))
    return torch.cat([f.cos(), f.sin()], dim=-1).contiguous().to(device)


class Rotary(NamedTuple):
    """A model's rotary positions, without a table of angles."""
    turns: torch.Tensor         # [rotary_dim / 2] fp64 on the device: revolutions per position
    amplitude: float = 1.0      # factor of the rotated dims
    adjacent: bool = False      # pairs (2 j, 2 j + 1) instead of (j, j + rotary_dim / 2)


def scaled_rotary(rotary_dim: int, theta: float = 500000.0, rule: str = "none",
                  factor: float = 1.0, original_max_position: int = 8192,
                  low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                  beta_fast: float = 32.0, beta_slow: float = 1.0, amplitude: float | None = None,
                  adjacent: bool = False, device="cpu") -> Rotary:
    """Frequencies theta^(-2 j / rotary_dim), scaled for contexts `factor` times as long by `rule`:

      none     as they are
      linear   all divided by factor
      ntk      theta grown so that the lowest frequency is divided by factor, the highest kept
      llama3   those of fewer than low_freq_factor revolutions in the original context divided,
               those of more than high_freq_factor kept, a mean of both between them
      yarn     the same between beta_slow and beta_fast revolutions, by a ramp over the dims' numbers,
               and an amplitude of 0.1 ln(factor) + 1
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim={rotary_dim} must be even and positive")
    if factor < 1:
        raise ValueError(f"factor={factor} must be at least 1")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if rule == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    w = theta ** (-i / rotary_dim)
    if rule == "linear":
        w = w / factor
    elif rule == "llama3":
        turns = original_max_position * w / (2 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0, 1)
        w = w / factor * (1 - keep) + w * keep
    elif rule == "yarn":
        lo, hi = (rotary_dim * math.log(original_max_position / (b * 2 * math.pi))
                  / (2 * math.log(theta)) for b in (beta_fast, beta_slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rotary_dim - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        w = w / factor * ramp + w * (1 - ramp)
        if amplitude is None:
            amplitude = 0.1 * math.log(factor) + 1
    elif rule not in ("none", "ntk"):
        raise ValueError(f"unknown scaling rule {rule!r}")
    return Rotary((w / (2 * math.pi)).to(device), 1.0 if amplitude is None else float(amplitude),
                  adjacent)
