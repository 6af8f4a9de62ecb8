"""Rotary positions: the table of a model's angles, as ``backend.rotary`` and
``backend.rotary_store`` take it.

The reference rotates queries and keys in its own layers before
Attention.forward stores and attends to them (nanovllm/layers/attention.py:
75-93); here the rotation joins the store.
"""
from __future__ import annotations

import math
from typing import Mapping, Sequence

import torch

from nanokv import _lib
from nanokv.paged_kv import ops

LAYOUTS = {"half": _lib.NKV_ROTARY_HALF, "interleaved": _lib.NKV_ROTARY_INTERLEAVED}
_SCALING_KEYS = {
    "linear": {"factor"},
    "ntk": {"factor"},
    "yarn": {"factor", "original_max_position", "fast_turns", "slow_turns", "attention_factor"},
    "bands": {"factor", "low_freq_factor", "high_freq_factor", "original_max_position"},
}
_OPTIONAL = {"fast_turns", "slow_turns", "attention_factor"}


def inverse_frequencies(rotary_dim: int, base: float = 10000.0,
                        scaling: Mapping | None = None) -> tuple[list[float], float]:
    """Radians per position of each of the rotary_dim / 2 pairs, base^(-2 j /
    rotary_dim) scaled for long contexts, and the factor of cosine and sine.

    ``scaling`` is None or a mapping with a ``type``:

    * ``linear``: positions divided by ``factor``;
    * ``ntk``: base times factor^(d / (d - 2)), which leaves the fastest pair
      as it is and divides the slowest by ``factor``;
    * ``yarn``: pairs that turn more than ``fast_turns`` (32) times within
      ``original_max_position`` positions keep their frequency, those under
      ``slow_turns`` (1) are divided by ``factor``, a linear ramp over the
      pair index in between; cosine and sine times ``attention_factor``
      (0.1 ln factor + 1 by default);
    * ``bands``: pairs with a wavelength under original_max_position /
      ``high_freq_factor`` keep their frequency, those over
      original_max_position / ``low_freq_factor`` are divided by ``factor``,
      linear in turns in between."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError("base must be finite and above 1")
    kind, factor = None, 1.0
    if scaling is not None:
        kind = scaling.get("type")
        keys = _SCALING_KEYS.get(kind)
        if keys is None:
            raise ValueError(f"rotary scaling type must be one of {sorted(_SCALING_KEYS)}, not {kind!r}")
        given = set(scaling) - {"type"}
        if not keys - _OPTIONAL <= given <= keys:
            raise ValueError(f"{kind} scaling takes {sorted(keys)}, not {sorted(given)}")
        for key in given:
            value = scaling[key]
            if value is None and key in _OPTIONAL:
                continue
            if not (math.isfinite(value) and value > 0):
                raise ValueError(f"rotary scaling {key} must be finite and positive")
        factor = float(scaling["factor"])
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = [base ** (-2.0 * j / rotary_dim) for j in range(rotary_dim // 2)]
    if kind == "linear":
        return [w / factor for w in inv], 1.0
    if kind == "yarn":
        original = float(scaling["original_max_position"])

        def index_of(turns: float) -> float:  # the pair that turns so often
            return rotary_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))

        low = max(math.floor(index_of(float(scaling.get("fast_turns") or 32.0))), 0)
        high = min(math.ceil(index_of(float(scaling.get("slow_turns") or 1.0))), rotary_dim - 1)
        out = []
        for j, w in enumerate(inv):
            ramp = min(1.0, max(0.0, (j - low) / max(high - low, 1e-3)))
            out.append(w / factor * ramp + w * (1.0 - ramp))
        attention = scaling.get("attention_factor")
        return out, float(attention) if attention is not None else 0.1 * math.log(factor) + 1.0
    if kind == "bands":
        slow, fast = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not fast > slow:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        original = float(scaling["original_max_position"])
        out = []
        for w in inv:
            smooth = min(1.0, max(0.0, (original * w / (2 * math.pi) - slow) / (fast - slow)))
            out.append(w * ((1.0 - smooth) / factor + smooth))
        return out, 1.0
    return inv, 1.0


class RotaryTable:
    """Cosines and sines of positions [0, max_position) for the first
    ``rotary_dim`` dims of each head, fp32 values of fp64 angles, on one GPU
    ([max_position, rotary_dim / 2, 2]; 512 bytes a position at 128 dims).

    ``layout``: pairs (j, j + rotary_dim / 2) ("half") or (2 j, 2 j + 1)
    ("interleaved").  ``sections``: how many pairs take their position from
    each of three rows (time, height, width; multimodal positions), None for
    one row.  ``inv_freq`` gives the radians per position themselves, in
    place of ``base`` and ``scaling``."""

    def __init__(self, rotary_dim: int, max_position: int, *, base: float = 10000.0,
                 layout: str = "half", scaling: Mapping | None = None,
                 sections: Sequence[int] | None = None, inv_freq: Sequence[float] | None = None,
                 device: torch.device | str = "cuda") -> None:
        if layout not in LAYOUTS:
            raise ValueError(f"rotary layout must be one of {sorted(LAYOUTS)}, not {layout!r}")
        if not 0 < int(max_position) <= 2**31 - 1:
            raise ValueError("max_position must be in [1, 2^31)")
        if rotary_dim < 2 or rotary_dim % 2:
            raise ValueError("rotary_dim must be even and positive")
        half = rotary_dim // 2
        if sections is not None:
            sections = tuple(int(n) for n in sections)
            if len(sections) != 3 or min(sections) < 0 or sum(sections) != half:
                raise ValueError("sections must be three counts of pairs that sum to rotary_dim / 2")
        if inv_freq is not None:
            if scaling is not None:
                raise ValueError("inv_freq and scaling exclude each other")
            frequencies, factor = [float(w) for w in inv_freq], 1.0
            if len(frequencies) != half or not all(math.isfinite(w) for w in frequencies):
                raise ValueError("inv_freq must hold rotary_dim / 2 finite values")
        else:
            frequencies, factor = inverse_frequencies(rotary_dim, float(base), scaling)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("RotaryTable requires a ROCm (cuda) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.rotary_dim = int(rotary_dim)
        self.max_position = int(max_position)
        self.layout = layout
        self.layout_code = LAYOUTS[layout]
        self.sections = sections
        self.section_ends = (half, half) if sections is None else (sections[0], sections[0] + sections[1])
        self.factor = factor
        self.inv_freq = frequencies
        self.table = ops.build_rotary_table(frequencies, factor, self.max_position, self.device)
