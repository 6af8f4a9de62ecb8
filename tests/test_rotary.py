"""Rotary frequencies against their formulas, and what the rotary entry points
and the page copies refuse, on the CPU (nothing here reaches a kernel)."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from nanokv import _lib
from nanokv.paged_kv import create_paged_kv_backend
from nanokv.paged_kv.hip_backend import validate_block_pairs
from nanokv.rotary import RotaryTable, inverse_frequencies


def test_plain_and_linear_and_ntk_frequencies():
    inv, factor = inverse_frequencies(8, 10000.0)
    assert factor == 1.0 and inv == [10000.0 ** (-j / 4) for j in range(4)]
    assert inverse_frequencies(8, 10000.0, {"type": "linear", "factor": 4})[0] == [w / 4 for w in inv]
    ntk = inverse_frequencies(8, 10000.0, {"type": "ntk", "factor": 4})[0]
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], inv[-1] / 4, rel_tol=1e-12)


def test_yarn_and_bands_keep_the_fast_pairs_and_divide_the_slow_ones():
    inv = inverse_frequencies(128, 1e6)[0]
    yarn, factor = inverse_frequencies(128, 1e6, {"type": "yarn", "factor": 8,
                                                  "original_max_position": 32768})
    assert math.isclose(factor, 0.1 * math.log(8) + 1)
    bands, one = inverse_frequencies(128, 1e6, {
        "type": "bands", "factor": 8, "low_freq_factor": 1, "high_freq_factor": 4,
        "original_max_position": 8192})
    assert one == 1.0
    for scaled in (yarn, bands):
        assert scaled[0] == inv[0] and math.isclose(scaled[-1], inv[-1] / 8, rel_tol=1e-12)
        ratios = [s / w for s, w in zip(scaled, inv)]
        assert all(a >= b - 1e-15 for a, b in zip(ratios, ratios[1:]))  # never less with slower pairs
        assert 0 < sum(1 / 8 < r < 1 for r in ratios) < 64
    # a pair whose wavelength lies half way between the bands, in turns
    turns = [8192 * w / (2 * math.pi) for w in inv]
    for w, s, n in zip(inv, bands, turns):
        if 1 < n < 4:
            share = (n - 1) / 3
            assert math.isclose(s, w * share + w / 8 * (1 - share), rel_tol=1e-12)
    given = inverse_frequencies(128, 1e6, {"type": "yarn", "factor": 8, "attention_factor": 1.5,
                                           "original_max_position": 32768})[1]
    assert given == 1.5


@pytest.mark.parametrize("dim,base,scaling,message", [
    (7, 1e4, None, "even"), (0, 1e4, None, "even"), (8, 1.0, None, "base"), (8, float("nan"), None, "base"),
    (8, 1e4, {"type": "other"}, "type"), (8, 1e4, {"type": "linear"}, "takes"),
    (8, 1e4, {"type": "linear", "factor": 0.0}, "positive"),
    (8, 1e4, {"type": "linear", "factor": 2, "extra": 1}, "takes"),
    (2, 1e4, {"type": "ntk", "factor": 2}, "one pair"),
    (8, 1e4, {"type": "bands", "factor": 2, "low_freq_factor": 4, "high_freq_factor": 4,
              "original_max_position": 64}, "above"),
])
def test_bad_frequencies_are_refused(dim, base, scaling, message):
    with pytest.raises(ValueError, match=message):
        inverse_frequencies(dim, base, scaling)


@pytest.mark.parametrize("kwargs,message", [
    (dict(layout="other"), "layout"), (dict(max_position=0), "max_position"),
    (dict(max_position=2**31), "max_position"), (dict(rotary_dim=9), "even"),
    (dict(sections=(1, 1)), "sections"), (dict(sections=(1, 1, 1)), "sections"),
    (dict(sections=(5, -1, 0)), "sections"), (dict(inv_freq=[1.0]), "rotary_dim / 2"),
    (dict(inv_freq=[1.0, 1.0, 1.0, float("inf")]), "finite"),
    (dict(inv_freq=[1.0] * 4, scaling={"type": "linear", "factor": 2}), "exclude"),
    (dict(device="cpu"), "ROCm"),
])
def test_bad_tables_are_refused(kwargs, message):
    arguments = {"rotary_dim": 8, "max_position": 16, **kwargs}
    with pytest.raises(ValueError, match=message):
        RotaryTable(arguments.pop("rotary_dim"), arguments.pop("max_position"), **arguments)


def desc(**changes) -> _lib.RotaryDesc:
    """A descriptor that is in order but for its pointers, which are null."""
    d = _lib.RotaryDesc()
    values = dict(num_tokens=4, num_q_heads=2, num_kv_heads=1, head_dim=64, rotary_dim=64,
                  max_position=16, q_token_stride=128, q_head_stride=64, k_token_stride=64,
                  k_head_stride=64, q_out_token_stride=128, q_out_head_stride=64,
                  k_out_token_stride=64, k_out_head_stride=64, position_bytes=8, dtype=1, **{})
    values.update(changes)
    ends = values.pop("section_ends", (32, 32))
    d.section_ends[0], d.section_ends[1] = ends
    for name, value in values.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=9), "dtype"), (dict(num_tokens=-1), "tokens"), (dict(num_tokens=2**31), "tokens"),
    (dict(num_q_heads=2000), "heads"), (dict(head_dim=0), "head_dim"), (dict(head_dim=2048), "head_dim"),
    (dict(rotary_dim=63), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(layout=2), "layout"), (dict(position_bytes=2), "positions"),
    (dict(max_position=0), "max_position"), (dict(position_row_stride=4, section_ends=(40, 20)), "sections"),
    (dict(position_row_stride=4, section_ends=(8, 40)), "sections"), (dict(num_slots=-1), "num_slots"),
    (dict(q_token_stride=-1), "stride"), (dict(), "null"), (dict(key_cache=4096, positions=4096), "null"),
])
def test_bad_rotary_descriptors_fail_before_launch(changes, message):
    library = _lib.load_library()
    assert library.nkv_rotary(ctypes.byref(desc(**changes)), None) != 0
    assert message in library.nkv_last_error().decode()


BASE = dict(q=0x10000, k=0x20000, q_out=0x30000, k_out=0x40000, positions=0x50000, table=0x60000)


@pytest.mark.parametrize("changes", [
    dict(q_out=0x10000 + 16),                        # a shifted input
    dict(q_out=0x10000, q_out_token_stride=64, q_out_head_stride=256),  # the input in another order
    dict(q_out=0x20000), dict(k_out=0x10000), dict(k_out=0x30000 + 128),  # another tensor's memory
    dict(q_out_token_stride=0), dict(q_out_head_stride=0), dict(q_out_head_stride=32),  # expanded
    dict(q_out_token_stride=96), dict(k_out_token_stride=32),
    dict(q=0x10000, k=0x10000 + 256, q_token_stride=192, k_token_stride=192, k_out=0x10000 + 128,
         k_out_token_stride=192),                    # in a fused row, but q's second head
    dict(k_out=0x20000, v=0x20000, v_token_stride=64, v_head_stride=64, key_cache=0x70000,
         value_cache=0x80000, slot_mapping=0x90000, num_slots=4),  # k's output over v
])
def test_overlapping_rotary_outputs_fail_before_launch(changes):
    library = _lib.load_library()
    assert library.nkv_rotary(ctypes.byref(desc(**{**BASE, **changes})), None) != 0
    assert "overlap" in library.nkv_last_error().decode()


def test_other_bad_calls_fail_before_launch():
    lib = _lib.load_library()
    assert lib.nkv_rotary(None, None) != 0 and "null" in lib.nkv_last_error().decode()
    for call, message in (
            (lambda: lib.nkv_rotary_table(None, 1.0, 4, 7, None, None), "even"),
            (lambda: lib.nkv_rotary_table(None, 1.0, 0, 8, None, None), "max_position"),
            (lambda: lib.nkv_rotary_table(None, 1.0, 4, 8, None, None), "null"),
            (lambda: lib.nkv_copy_blocks(None, None, -1, 4, 4, 64, None, 1, None), "negative"),
            (lambda: lib.nkv_copy_blocks(None, None, 1, 4, 4, 64, None, 1, None), "null"),
            (lambda: lib.nkv_copy_blocks(64, 64, 1, 4, 4, 64, 4, 1, None), "8-byte"),
            (lambda: lib.nkv_copy_blocks(64, 64, 70000, 4, 4, 64, 64, 1, None), "too many"),
            (lambda: lib.nkv_copy_blocks(64, 64, 1, 4, 4, 8192, 64, 2**31, None), "too many"),
            (lambda: lib.nkv_copy_blocks(64, 64, 1, 4, 4, 8192, 64, 2**24, None), "too many"),
            (lambda: lib.nkv_copy_blocks(65, 64, 1, 4, 4, 64, 64, 1, None), "aligned"),
            (lambda: lib.nkv_pool_apply_log(None, None, 1, None, 0, None, 0, None), "null pool"),
            (lambda: lib.nkv_pool_apply_copies(None, None, 1, None, 0, None, 0, None), "null pool")):
        assert call() != 0
        assert message in lib.nkv_last_error().decode(), message
    assert lib.nkv_copy_blocks(None, None, 1, 4, 4, 64, None, 0, None) == 0  # nothing to do


def test_block_pair_rules():
    def check(pairs, same=True, src=8, dst=8):
        validate_block_pairs(torch.tensor(pairs, dtype=torch.int32).reshape(-1, 2), src, dst, same=same)

    check([(0, 4), (0, 5), (1, 6), (3, 3)])
    check([(0, 1), (1, 2)], same=False)
    for pairs, message in (([(8, 1)], "outside"), ([(0, -1)], "outside"), ([(0, 1), (2, 1)], "twice"),
                           ([(0, 1), (1, 2)], "source")):
        with pytest.raises(ValueError, match=message):
            check(pairs)


def test_the_backend_refuses_host_tensors():
    backend = create_paged_kv_backend("hip")
    cache = torch.zeros(2, 3, 4, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device"):
        backend.copy_blocks(cache, [(0, 1)])
    with pytest.raises(ValueError, match="outside"):
        backend.copy_blocks(cache, [(0, 3)])
    with pytest.raises(ValueError, match="twice"):
        backend.copy_blocks(cache, [(0, 1), (2, 1)])
