"""Tables of rotary positions: cosines and sines in fp32 from 64-bit angles, plain or scaled for contexts longer than the
one a model was trained on.  `ops.rotary` and `ops.kv_append` apply them (pairs (i, i + R/2), or (2i, 2i+1) when interleaved)."""
import math

import torch


# What a dict of each type may hold besides "rope_type" / "type", "rope_theta" and "partial_rotary_factor".
_KEYS = {
    "default": (),
    "linear": ("factor",),
    "ntk": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
    "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale",
             "mscale_all_dim"),
}


def _scaling(scaling, base):
    """(type, base, the other keys that are set) of a dict of scaling; refuses what it does not know: a key that is left out of account
    would make another model's table."""
    given = {k: v for k, v in scaling.items() if v is not None}
    kinds = {given.pop(k) for k in ("rope_type", "type") if k in given}
    kind = kinds.pop() if len(kinds) == 1 else None
    if kind not in _KEYS:
        raise ValueError(f"rotary_frequencies: scaling must name one type of {', '.join(_KEYS)}, got {scaling}")
    theta = given.pop("rope_theta", None)
    if theta is not None and base is not None and float(theta) != float(base):
        raise ValueError(f"rotary_frequencies: base {base} and the scaling's rope_theta {theta} differ")
    if float(given.pop("partial_rotary_factor", 1.0)) != 1.0:
        raise ValueError("rotary_frequencies: rotary_dim is the part of a head that turns; apply the scaling's partial_rotary_factor "
                         f"to it and leave it out, got {scaling}")
    unknown = sorted(set(given) - set(_KEYS[kind]))
    if unknown:
        raise ValueError(f"rotary_frequencies: a scaling of type {kind} may hold {', '.join(_KEYS[kind]) or 'nothing else'}; not known: "
                         f"{', '.join(unknown)}")
    return kind, theta if base is None else base, given


def _number(given, name, default=None):
    """A positive number of the scaling."""
    v = given.get(name, default)
    if v is None or isinstance(v, (bool, str)) or not 0.0 < float(v) < math.inf:
        raise ValueError(f"rotary_frequencies: the scaling needs {name}, a positive number, got {v!r}")
    return float(v)


def rotary_frequencies(rotary_dim, base=None, scaling=None):
    """(frequencies fp64 [rotary_dim / 2], gain): position p turns pair i by p * frequencies[i]; cosines and sines are
    multiplied by gain.  base: 10000 unless it or the scaling's "rope_theta" is given.  scaling: None, or a dict in the form of a model
    configuration's `rope_scaling` or `rope_parameters`, by its "rope_type" (or "type"):
      default  no scaling
      linear   every frequency divided by `factor`
      ntk      the base multiplied by factor^(R / (R - 2))
      llama3   wavelengths over original / low_freq_factor divided by `factor`, those under original / high_freq_factor kept,
               a linear ramp over the turns made within the original length in between
      yarn     pairs that turn more than beta_fast (32) times within the original length kept, those that turn less than beta_slow (1)
               divided by `factor`, a linear ramp over the pairs' indices in between, whose ends are whole pairs unless "truncate" is false;
               gain: attention_factor, else g(mscale) / g(mscale_all_dim) where both are given, else g(1), g(m) = 0.1 m ln(factor) + 1
    with the original length in "original_max_position_embeddings".  A key that the type does not know raises ValueError."""
    R = int(rotary_dim)
    if R <= 0 or R % 16:
        raise ValueError(f"rotary_frequencies: rotary_dim must be a positive multiple of 16, got {rotary_dim}")
    kind, given = "default", {}
    if scaling is not None:
        kind, base, given = _scaling(scaling, base)
    base = 10000.0 if base is None else float(base)
    if not base > 1.0:
        raise ValueError(f"rotary_frequencies: base must be above 1, got {base}")
    power = torch.arange(0, R, 2, dtype=torch.float64) / R
    freq = base ** -power
    if kind == "default":
        return freq, 1.0
    factor = _number(given, "factor")
    if not factor >= 1.0:
        raise ValueError(f"rotary_frequencies: the scaling's factor must be at least 1, got {scaling}")
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        return (base * factor ** (R / (R - 2.0))) ** -power, 1.0
    original = _number(given, "original_max_position_embeddings")
    turns = original * freq / (2.0 * math.pi)                     # of each pair within the original length
    if kind == "llama3":
        low, high = _number(given, "low_freq_factor"), _number(given, "high_freq_factor")
        if not high > low:
            raise ValueError(f"rotary_frequencies: high_freq_factor must be above low_freq_factor, got {scaling}")
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return freq * (keep + (1.0 - keep) / factor), 1.0

    fast, slow = _number(given, "beta_fast", 32.0), _number(given, "beta_slow", 1.0)
    truncate = given.get("truncate", True)
    if not fast > slow or not isinstance(truncate, bool):
        raise ValueError(f"rotary_frequencies: beta_fast must be above beta_slow and truncate True or False, got {scaling}")
    # the pairs that turn so often within the original length
    first, last = (R * math.log(original / (n * 2.0 * math.pi)) / (2.0 * math.log(base)) for n in (fast, slow))
    if truncate:
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, R - 1)
    ramp = ((torch.arange(R // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
    if "attention_factor" in given:
        gain = _number(given, "attention_factor")
    elif "mscale" in given or "mscale_all_dim" in given:          # one alone has been read in more than one way: refused
        gain = (0.1 * _number(given, "mscale") * math.log(factor) + 1.0) / (0.1 * _number(given, "mscale_all_dim") * math.log(factor) + 1.0)
    else:
        gain = 0.1 * math.log(factor) + 1.0
    return freq * (1.0 - ramp + ramp / factor), gain


def rotary_table(max_positions, rotary_dim, base=None, scaling=None, device="cuda"):
    """fp32 [max_positions, rotary_dim / 2, 2] of (cosine, sine) for positions 0 .. max_positions - 1.  Angles are formed and
    reduced in 64 bits: at position 10^6 a 32-bit angle is off by 0.06 radians.  512 bytes a position at rotary_dim 128."""
    if int(max_positions) <= 0:
        raise ValueError(f"rotary_table: max_positions must be positive, got {max_positions}")
    freq, gain = rotary_frequencies(rotary_dim, base, scaling)
    angle = torch.arange(int(max_positions), dtype=torch.float64, device=device)[:, None] * freq.to(device)[None, :]
    return torch.stack((torch.cos(angle) * gain, torch.sin(angle) * gain), dim=-1).float().contiguous()
