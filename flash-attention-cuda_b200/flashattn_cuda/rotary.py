"""Frequencies of rotary positions, for rope() and append_paged()."""

import math

import torch


def rope_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0,
                     original_length=None, low=1.0, high=None, device="cuda"):
    """Radians that one position turns each of the rotary_dim / 2 pairs by,
    as float64 on `device`, and the amplitude to pass beside them.

    Pair i turns by base ** (-2 i / rotary_dim). `scaling` stretches that for
    a context `factor` times as long as the model was trained on:

    - None: as it is;
    - "linear": every frequency divided by `factor` (positions interpolated);
    - "base": base * factor ** (d / (d - 2)) in the place of base, which
      leaves the fastest pair alone and divides the slowest by `factor`;
    - "bands": by how often a pair turns over the `original_length` positions
      of training: `low` (1) times or fewer, divided by `factor`; `high` (4)
      times or more, left alone; between, the two mixed linearly in that
      number;
    - "yarn": as "bands" with the mix linear in the pair's index and `high`
      32, and an amplitude of 0.1 ln(factor) + 1 (Peng et al., YaRN, 2023).
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError(f"base must be finite and above 1, got {base}")
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"factor must be finite and at least 1, got {factor}")
    if scaling == "base":
        if rotary_dim < 4:
            raise ValueError("base scaling needs a rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freqs = base ** (-2.0 * pair / rotary_dim)
    amplitude = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling in ("bands", "yarn"):
        if not original_length or original_length <= 0:
            raise ValueError(f"{scaling} scaling needs original_length")
        if high is None:
            high = 4.0 if scaling == "bands" else 32.0
        if not 0.0 < low < high:
            raise ValueError(f"low and high must be 0 < low < high, got {low} and {high}")
        if scaling == "bands":
            keep = (freqs * original_length / (2.0 * math.pi) - low) / (high - low)
        else:
            def index(turns):  # of the pair that turns so often
                return (rotary_dim * math.log(original_length / (2.0 * math.pi * turns))
                        / (2.0 * math.log(base)))
            first = max(math.floor(index(high)), 0)
            last = min(math.ceil(index(low)), rotary_dim - 1)
            keep = 1.0 - (pair - first) / max(last - first, 1e-3)
            amplitude = 0.1 * math.log(factor) + 1.0
        keep = keep.clamp(0.0, 1.0)
        freqs = freqs * keep + freqs / factor * (1.0 - keep)
    elif scaling not in (None, "base"):
        raise ValueError("scaling must be None, 'linear', 'base', 'bands' or "
                         f"'yarn', got {scaling!r}")
    return freqs.to(device), amplitude
