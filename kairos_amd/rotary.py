"""Tables of rotary positions: cosines and sines in fp32 from 64-bit angles, plain or scaled for contexts longer than the
one a model was trained on.  `ops.rotary` and `ops.kv_append` apply them (pairs (i, i + R/2), or (2i, 2i+1) when interleaved)."""
import math

import torch


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None):
    """(frequencies fp64 [rotary_dim / 2], gain): position p turns pair i by p * frequencies[i]; cosines and sines are
    multiplied by gain.  scaling: None, or a dict in the form of a model configuration's `rope_scaling`, by its "rope_type"
    (or "type"):
      linear   every frequency divided by `factor`
      ntk      the base multiplied by factor^(R / (R - 2))
      llama3   wavelengths over original / low_freq_factor divided by `factor`, those under original / high_freq_factor kept,
               a linear ramp over the turns made within the original length in between
      yarn     pairs that turn more than beta_fast (32) times within the original length kept, those that turn less than beta_slow (1)
               divided by `factor`, a linear ramp over the pairs' indices in between; gain 0.1 ln(factor) + 1 (attention_factor)
    with the original length in "original_max_position_embeddings"."""
    R = int(rotary_dim)
    if R <= 0 or R % 16:
        raise ValueError(f"rotary_frequencies: rotary_dim must be a positive multiple of 16, got {rotary_dim}")
    if not base > 1.0:
        raise ValueError(f"rotary_frequencies: base must be above 1, got {base}")
    power = torch.arange(0, R, 2, dtype=torch.float64) / R
    freq = float(base) ** -power
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type"))
    if kind == "default":
        return freq, 1.0
    factor = float(scaling.get("factor", 0.0))
    if kind not in ("linear", "ntk", "llama3", "yarn") or not factor >= 1.0:
        raise ValueError(f"rotary_frequencies: scaling must be linear, ntk, llama3 or yarn with a factor >= 1, got {scaling}")
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        return (float(base) * factor ** (R / (R - 2.0))) ** -power, 1.0
    original = float(scaling["original_max_position_embeddings"])
    turns = original * freq / (2.0 * math.pi)                     # of each pair within the original length
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low:
            raise ValueError(f"rotary_frequencies: high_freq_factor must be above low_freq_factor, got {scaling}")
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return freq * (keep + (1.0 - keep) / factor), 1.0

    def index_of(n):                                              # the pair that makes n turns within the original length
        return R * math.log(original / (n * 2.0 * math.pi)) / (2.0 * math.log(float(base)))

    first = max(math.floor(index_of(float(scaling.get("beta_fast") or 32.0))), 0)
    last = min(math.ceil(index_of(float(scaling.get("beta_slow") or 1.0))), R - 1)
    ramp = ((torch.arange(R // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
    gain = scaling.get("attention_factor")
    return freq * (1.0 - ramp + ramp / factor), float(gain) if gain is not None else 0.1 * math.log(factor) + 1.0


def rotary_table(max_positions, rotary_dim, base=10000.0, scaling=None, device="cuda"):
    """fp32 [max_positions, rotary_dim / 2, 2] of (cosine, sine) for positions 0 .. max_positions - 1.  Angles are formed and
    reduced in 64 bits: at position 10^6 a 32-bit angle is off by 0.06 radians.  512 bytes a position at rotary_dim 128."""
    if int(max_positions) <= 0:
        raise ValueError(f"rotary_table: max_positions must be positive, got {max_positions}")
    freq, gain = rotary_frequencies(rotary_dim, base, scaling)
    angle = torch.arange(int(max_positions), dtype=torch.float64, device=device)[:, None] * freq.to(device)[None, :]
    return torch.stack((torch.cos(angle) * gain, torch.sin(angle) * gain), dim=-1).float().contiguous()
