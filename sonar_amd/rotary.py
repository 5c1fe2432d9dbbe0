"""Tables of cosines and sines that `ops.qk_norm_rope` and `ops.qk_norm_rope_append` read: made once, at load."""
from __future__ import annotations

import math

import torch


#: The numbers that each kind of scaling needs, and those that it may have.
_NUMBERS = {"default": ((), ()), "linear": (("factor",), ()),
            "llama3": (("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"), ()),
            "yarn": (("factor", "original_max_position_embeddings"),
                     ("beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"))}
#: What may stand beside them and changes no table: that of `base` has to agree, the other is in rotary_dim.
_BESIDE = ("rope_type", "type", "rope_theta", "partial_rotary_factor", "original_max_position_embeddings")


def _checked(scaling: dict | None, base: float) -> dict:
    """The kind of a scaling and its numbers, those that are None left out; ValueError where something is missing or not known."""
    if scaling is None:
        return {"rope_type": "default"}
    scaling = {name: value for name, value in scaling.items() if value is not None}
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind not in _NUMBERS or scaling.get("type", kind) != kind:
        raise ValueError(f"rope_type = {kind!r} (type = {scaling.get('type')!r}) is not one of {', '.join(_NUMBERS)}")
    needed, possible = _NUMBERS[kind]
    missing, unknown = set(needed) - set(scaling), set(scaling) - {*needed, *possible, *_BESIDE}
    if missing or unknown:
        raise ValueError(f"a scaling of rope_type {kind!r} without {sorted(missing)}" if missing else
                         f"a scaling of rope_type {kind!r} with {sorted(unknown)}, which it does not take")
    if scaling.get("rope_theta", base) != base:
        raise ValueError(f"rope_theta = {scaling['rope_theta']} and base = {base}")
    if not scaling.get("factor", 1.0) > 0:
        raise ValueError(f"factor = {scaling['factor']} must be positive")
    return {**scaling, "rope_type": kind}


def rotary_rates(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> torch.Tensor:
    """The angle of each pair per position, float64 (rotary_dim / 2,): base ** (-2 i / rotary_dim), and with `scaling`, as a model's
    configuration holds it ("rope_type" and its numbers; a number that this function does not know is refused, not left out):

      default  as without
      linear   every rate divided by `factor`
      llama3   by wavelength: those longer than original_max_position_embeddings / low_freq_factor are divided by `factor`, those
               shorter than it / high_freq_factor stay, a straight line of the inverse wavelength between
      yarn     by turns within original_max_position_embeddings: pairs of `beta_fast` (32) turns or more stay, of `beta_slow` (1) or
               fewer are divided by `factor`, a straight line of the pair's number between, whose ends are whole pairs unless
               `truncate` is false"""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim = {rotary_dim} must be even and positive")
    rates = float(base) ** -(torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    scaling = _checked(scaling, base)
    kind = scaling["rope_type"]
    if kind == "default":
        return rates
    factor = float(scaling["factor"])
    if kind == "linear":
        return rates / factor
    original = scaling["original_max_position_embeddings"]
    if kind == "llama3":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        stay = ((rates * original / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
    else:
        # the pair that turns n times within the original context
        pair = lambda n: rotary_dim * math.log(original / (2 * math.pi * n)) / (2 * math.log(base))  # noqa: E731
        first, last = pair(scaling.get("beta_fast", 32)), pair(scaling.get("beta_slow", 1))
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rotary_dim - 1)
        stay = 1 - ((torch.arange(rotary_dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0, 1)
    return rates * stay + rates / factor * (1 - stay)


def _yarn_size(scaling: dict) -> float:
    """What yarn multiplies cosines and sines by."""
    factor = scaling["factor"]
    if scaling.get("attention_factor"):
        return scaling["attention_factor"]
    size = lambda m: 0.1 * m * math.log(factor) + 1 if factor > 1 else 1.0  # noqa: E731
    queries, keys = scaling.get("mscale"), scaling.get("mscale_all_dim")
    if queries and keys:
        return size(queries) / size(keys)
    if keys or (queries or 1) != 1:   # (what one of them alone stands for is not agreed)
        raise ValueError(f"mscale = {queries} and mscale_all_dim = {keys} go together")
    return size(1.0)


def rotary_cos_sin(rotary_dim: int, max_position: int, base: float = 10000.0, scaling: dict | None = None,
                   device: torch.device | str | None = None) -> torch.Tensor:
    """float32 (max_position, rotary_dim): a position's cosines, then its sines.  The angles are formed in 64 bits, as those of far
    positions need; for yarn both are multiplied by `attention_factor`, and if the configuration does not say that, by
    (0.1 mscale ln(factor) + 1) / (0.1 mscale_all_dim ln(factor) + 1), or 0.1 ln(factor) + 1 without those."""
    angles = torch.arange(max_position, dtype=torch.float64)[:, None] * rotary_rates(rotary_dim, base, scaling)
    scaling = _checked(scaling, base)
    size = _yarn_size(scaling) if scaling["rope_type"] == "yarn" else 1.0
    return (torch.cat([angles.cos(), angles.sin()], dim=1) * size).float().to(device)
