"""Rotary positions for the rope parts of queries and keys.

The caches take the rope key, and the attention the rope query, as already rotated.
``apply_rotary`` rotates both in one launch, from where the projections leave them
to where they are used:

    rope = Rotary(64, base=10000.0, scaling={"type": "yarn", "factor": 40, ...}, device=dev)
    apply_rotary(rope, positions, q[..., 128:], k_pe, q_out=q_absorbed[..., 512:], k_out=k_rot)

Angles are exact for positions of any size: a pair's frequency is held as a 64-bit
fraction of a turn (FP32 angles are off by up to 2^-8 at position 10^5). Frequencies
follow the ``rope_scaling`` entry of a model's configuration; the reference leaves
this step to the model's own code.
"""

from __future__ import annotations

import math
from fractions import Fraction

import torch

from . import kernels

# 1 / (2 pi) to 64 digits: turns of a radian
_PER_TURN = Fraction("0.1591549430918953357688837633725143620344596457404564487476673441")


# what a scaling of each kind may state (besides the rotary base, where it is ``base``)
_STATED = {
    "default": (),
    "linear": ("factor", "original_max_position_embeddings"),
    "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "truncate", "mscale", "mscale_all_dim",
             "attention_factor"),
    "longrope": ("factor", "original_max_position_embeddings", "long_factor", "short_factor", "long", "attention_factor"),
}


def _yarn_ramp(dim, base, original, beta_fast, beta_slow, truncate):
    """0 for pairs that turn more than ``beta_fast`` times over the ``original`` length, 1 for those that turn
    less than ``beta_slow`` times, linear in the pair's number between (``truncate``: between whole numbers)."""

    def pair(turns):
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = pair(beta_fast), pair(beta_slow)
    if truncate:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    width = high - low if high > low else 0.001
    return [min(max((i - low) / width, 0.0), 1.0) for i in range(dim // 2)]


def frequencies(dim: int, base: float = 10000.0, scaling: dict | None = None):
    """``(angles, scale)``: the angle in radians of a step of one position for each of the ``dim / 2`` pairs, and the
    factor of sines and cosines.

    ``scaling``: a configuration's ``rope_scaling`` (its kind under ``type`` or ``rope_type``): ``linear``
    (``factor``), ``yarn`` (``factor``, ``original_max_position_embeddings``, ``beta_fast``, ``beta_slow``, ``truncate``, and
    ``mscale`` / ``mscale_all_dim`` or ``attention_factor``), ``longrope`` (``long_factor`` and ``short_factor``, a
    divisor for each pair, ``factor`` and ``original_max_position_embeddings``, or ``attention_factor``; ``long`` says
    which of the two lists, the first by default), ``default`` or None. An entry that its kind does not have, or one
    that is missing, is refused: configurations that keep the context's factor or original length outside of
    ``rope_scaling`` have to add them. Entries of None count as missing.
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary width must be even and positive, got {dim}")
    if not (math.isfinite(base) and base > 1):
        raise ValueError(f"rotary base must be finite and above 1, got {base}")
    f = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    s = {k: v for k, v in (scaling or {}).items() if v is not None}
    kind = s.get("type", s.get("rope_type", "default"))
    if kind not in _STATED:
        raise ValueError(f"unknown rope scaling {kind!r}")
    unknown = sorted(set(s) - {"type", "rope_type", "rope_theta", *_STATED[kind]})
    if unknown:
        raise ValueError(f"rope scaling {kind!r} has no {', '.join(unknown)}")
    if s.get("rope_theta", base) != base:
        raise ValueError(f"rope scaling states rope_theta {s['rope_theta']!r}, base is {base!r}")
    if kind == "default":
        return f, 1.0

    def number(key, default=None, least=0.0):
        v = s.get(key, default)
        if not isinstance(v, (int, float)) or not math.isfinite(v) or v <= least:
            raise ValueError(f"rope scaling {kind!r} needs {key} above {least}, got {v!r}")
        return float(v)

    if kind == "linear":
        factor = number("factor")
        return [x / factor for x in f], 1.0
    if kind == "yarn":
        factor, original = number("factor"), number("original_max_position_embeddings")
        ramp = _yarn_ramp(dim, base, original, number("beta_fast", 32.0), number("beta_slow", 1.0),
                          s.get("truncate", True))

        def mscale(m):
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

        by_m, by_all = s.get("mscale"), s.get("mscale_all_dim")
        if "attention_factor" in s:
            scale = number("attention_factor")
        elif by_m and by_all:
            scale = mscale(number("mscale")) / mscale(number("mscale_all_dim"))
        elif by_all or (by_m and by_m != 1):
            # (published code differs in what the other one is then)
            raise ValueError("rope scaling 'yarn' needs mscale and mscale_all_dim together, or attention_factor")
        else:
            scale = mscale(1.0)
        return [x / factor * r + x * (1.0 - r) for x, r in zip(f, ramp)], scale
    by = s.get("long_factor" if s.get("long", True) else "short_factor")
    if not isinstance(by, (list, tuple)) or len(by) != dim // 2 or not all(
            isinstance(v, (int, float)) and math.isfinite(v) and v > 0 for v in by):
        raise ValueError(f"rope scaling 'longrope' needs {dim // 2} positive factors")
    if "attention_factor" in s:
        scale = number("attention_factor")
    else:
        factor, original = number("factor"), number("original_max_position_embeddings", least=1.0)
        scale = math.sqrt(1.0 + math.log(factor) / math.log(original)) if factor > 1 else 1.0
    return [x / v for x, v in zip(f, by)], scale


class Rotary:
    """A model's rotary positions: width, layout, frequencies.

    ``interleaved``: pairs are elements (2 i, 2 i + 1) of a head, else (i, i + dim / 2). ``scaling`` as for
    :func:`frequencies`; or ``inv_freq``, the pairs' angles in radians (any floating sequence or tensor), and ``scale``
    directly. ``scale`` multiplies sines and cosines; a model's further factor on its logits stays with its ``sm_scale``.
    """

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = True, scaling: dict | None = None,
                 device="cuda", inv_freq=None, scale: float = 1.0):
        if dim > 512:
            raise ValueError(f"rotary width must be 512 at most, got {dim}")
        if inv_freq is None:
            angles, by = frequencies(dim, base, scaling)
        else:
            if scaling is not None:
                raise ValueError("give inv_freq or scaling, not both")
            if dim < 2 or dim % 2:
                raise ValueError(f"rotary width must be even and positive, got {dim}")
            angles = inv_freq.double().tolist() if isinstance(inv_freq, torch.Tensor) else [float(v) for v in inv_freq]
            by = 1.0
            if len(angles) != dim // 2 or not all(math.isfinite(v) for v in angles):
                raise ValueError(f"inv_freq must be {dim // 2} finite angles")
        self.dim = int(dim)
        self.interleaved = bool(interleaved)
        self.scale = float(scale) * by
        if not math.isfinite(self.scale):
            raise ValueError("rotary scale must be finite")
        self.inv_freq = angles
        # turns of a step, modulo one, times 2^64 (as the bits of an int64)
        turns = [round(Fraction(v) * _PER_TURN * 2**64) % 2**64 for v in angles]
        self.turns = torch.tensor([t - 2**64 if t >= 2**63 else t for t in turns], dtype=torch.int64, device=device)


def apply_rotary(rope: Rotary, positions, q, k=None, q_out=None, k_out=None):
    """Rotate ``q`` and ``k`` by ``positions``; returns ``(q_out, k_out)`` (``k_out`` None without ``k``).

    ``q``, ``k``: bf16, fp16 or fp32, ``[T, heads, dim]`` or ``[T, dim]`` views of any strides with a contiguous last dim
    (a part of a head is a slice of it). ``positions``: ``[T]``, any integers, negative ones turn back. Outputs of
    the same shapes receive the results; without one the tensor is rotated in place. An output is its input or does not
    overlap any input. One launch, FP32 arithmetic, one rounding.
    """
    if positions.dtype != torch.int64 or not positions.is_contiguous():
        if positions.dtype.is_floating_point or positions.dtype == torch.bool:
            raise TypeError(f"positions must be integers, got {positions.dtype}")
        positions = positions.to(torch.int64).contiguous()
    q_out = q if q_out is None else q_out
    if k is None:
        if k_out is not None:
            raise ValueError("k_out is given without k")
    elif k_out is None:
        k_out = k
    kernels.rotary(positions, rope.turns, rope.scale, rope.interleaved, q, q_out, k, k_out)
    return q_out, k_out
