"""Rotary positions on the GPU against the formula in 64 bits.

Bound of each element (x1, x2 its pair's inputs, f the scaling's factor): cosine
and sine are rounded to fp32, as are two products (or one, fused) and the
sum, each by 2^-24 relative to at most f (|x1| + |x2|): together under
d = 2^-22 f (|x1| + |x2|).  The result is rounded once more, by eps / 2 of
its value (fp16: at least 2^-25 below its normal range).
"""
from __future__ import annotations

import pytest
import torch

from nanokv.packing import capture_graph
from nanokv.rotary import RotaryTable

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def backend(gpu_device):
    from nanokv.paged_kv import create_paged_kv_backend

    return create_paged_kv_backend("hip")


def turned(x, positions, table):
    """(x rotated, the bound's d) in 64 bits on the CPU; positions [T] or [3, T]."""
    x = x.detach().cpu().double()
    p = positions.cpu().double()
    half = table.rotary_dim // 2
    p = p.expand(3, -1) if p.ndim == 1 else p
    e0, e1 = table.section_ends
    angle = torch.stack([p[0 if j < e0 else 1 if j < e1 else 2] * table.inv_freq[j]
                         for j in range(half)], 1)[:, None]
    if table.layout == "half":
        i1, i2 = slice(0, half), slice(half, 2 * half)
    else:
        i1, i2 = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    out, d = x.clone(), torch.zeros_like(x)
    c, s = angle.cos() * table.factor, angle.sin() * table.factor
    out[..., i1] = x[..., i1] * c - x[..., i2] * s
    out[..., i2] = x[..., i2] * c + x[..., i1] * s
    d[..., i1] = d[..., i2] = 2.0 ** -22 * table.factor * (x[..., i1].abs() + x[..., i2].abs())
    return out, d


def check(got, expected, what):
    ref, d = expected
    step = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    err = (got.cpu().double() - ref).abs()
    bound = torch.where(d > 0, d + step * (ref.abs() + d) + tiny, 0.0)  # other dims are copied
    assert bool((err <= bound).all()), f"{what}: worst {float((err - bound).max()):.3e} over the bound"


def heads(gen, device, tokens, dtype, q, kv, dim):
    fused = torch.randn(tokens, (q + 2 * kv) * dim, generator=gen).to(dtype).to(device)
    parts = fused.split([q * dim, kv * dim, kv * dim], 1)
    return [p.unflatten(1, (n, dim)) for p, n in zip(parts, (q, kv, kv))]


CASES = [
    # dtype, layout, head_dim, rotary_dim, sections, q heads, kv heads, tokens
    ("bf16", "half", 128, 128, None, 16, 8, 64),
    ("bf16", "half", 128, 128, (16, 24, 24), 28, 4, 1511),
    ("bf16", "half", 128, 128, (5, 30, 29), 16, 2, 77),  # sections inside a thread's pairs
    ("fp16", "interleaved", 128, 64, None, 16, 2, 300),
    ("fp32", "half", 128, 32, None, 4, 1, 129),
    ("fp32", "interleaved", 64, 64, (8, 12, 12), 3, 3, 33),
    ("bf16", "interleaved", 256, 128, None, 8, 1, 5),
    ("fp16", "half", 80, 20, None, 5, 5, 19),  # single elements
    ("bf16", "interleaved", 33, 32, None, 2, 1, 9),  # an odd dim at the end
    ("bf16", "half", 2, 2, None, 1, 1, 3),
    ("fp16", "half", 1024, 1024, None, 2, 1, 3),
    ("bf16", "half", 64, 64, (0, 0, 32), 40, 8, 1),
    ("bf16", "half", 128, 128, None, 28, 4, 5000),  # a thread walks several heads
    ("fp32", "interleaved", 96, 48, None, 32, 8, 2500),
]


@pytest.mark.parametrize("dtype,layout,dim,rot,sections,q_heads,kv_heads,tokens", CASES)
def test_rotary_and_rotary_store_match_the_formula(backend, gpu_device, dtype, layout, dim, rot,
                                                   sections, q_heads, kv_heads, tokens):
    gen = torch.Generator().manual_seed(tokens + dim + rot)
    table = RotaryTable(rot, 4096, base=10000.0, layout=layout, sections=sections, device=gpu_device,
                        scaling={"type": "yarn", "factor": 4.0, "original_max_position": 1024})
    q, k, v = heads(gen, gpu_device, tokens, DTYPES[dtype], q_heads, kv_heads, dim)
    shape = (3, tokens) if sections else (tokens,)
    positions = torch.randint(0, 4096, shape, generator=gen).to(gpu_device)
    ref_q, ref_k = turned(q, positions, table), turned(k, positions, table)
    for index_type in (torch.int64, torch.int32):
        got_q, got_k = backend.rotary(q, k, positions.to(index_type), table)
        check(got_q, ref_q, "q")
        check(got_k, ref_k, "k")
    # The store: -1 and slots past the cache are not stored, other rows stay.
    bs = 16
    nb = -(-2 * tokens // bs) + 1
    slots = torch.randperm(nb * bs, generator=gen)[:tokens].to(torch.int32)
    slots[::7] = -1
    if tokens > 3:
        slots[3] = nb * bs
    kc = torch.randn(nb, bs, kv_heads, dim, generator=gen).to(DTYPES[dtype]).to(gpu_device)
    vc = torch.randn(nb, bs, kv_heads, dim, generator=gen).to(DTYPES[dtype]).to(gpu_device)
    old_k, old_v = kc.clone(), vc.clone()
    k_out = torch.empty(k.shape, dtype=k.dtype, device=gpu_device)
    out = backend.rotary_store(q, k, v, kc, vc, slots.to(gpu_device), positions, table, k_out=k_out)
    assert torch.equal(out, got_q) and torch.equal(k_out, got_k)
    stored = (slots >= 0) & (slots < nb * bs)
    at = slots[stored].long().to(gpu_device)
    old_k.view(-1, kv_heads, dim)[at] = got_k[stored.to(gpu_device)]
    old_v.view(-1, kv_heads, dim)[at] = v[stored.to(gpu_device)]
    assert torch.equal(kc, old_k) and torch.equal(vc, old_v)


def test_in_place_strided_and_text_positions(backend, gpu_device):
    """q and k rotated where they lie; heads cut out of wider ones; a row of
    positions for a table with sections; three equal rows by expand()."""
    gen = torch.Generator().manual_seed(3)
    table = RotaryTable(64, 100, sections=(10, 11, 11), device=gpu_device)
    q, k, _ = heads(gen, gpu_device, 21, torch.bfloat16, 4, 2, 128)
    before = q.clone(), k.clone()
    positions = torch.arange(21, device=gpu_device) * 4
    ref = [turned(x[:, :, 8:72], positions, table) for x in before]
    wide_q, wide_k = backend.rotary(q[:, :, 8:72], k[:, :, 8:72], positions, table)
    check(wide_q, ref[0], "q view")
    check(wide_k, ref[1], "k view")
    again = backend.rotary(q[:, :, 8:72], k[:, :, 8:72], positions.expand(3, -1), table)
    assert torch.equal(again[0], wide_q) and torch.equal(again[1], wide_k)
    odd = backend.rotary(q[:, :, 5:69], k[:, :, 5:69], positions, table)  # 2-byte aligned views
    check(odd[0], turned(before[0][:, :, 5:69], positions, table), "odd view")
    inside = q[:, :, 8:72], k[:, :, 8:72]
    got = backend.rotary(*inside, positions, table, out=inside)
    assert got[0].data_ptr() == inside[0].data_ptr()
    assert torch.equal(inside[0], wide_q) and torch.equal(inside[1], wide_k)
    for x, old in zip((q, k), before):  # the dims around the view
        assert torch.equal(x[:, :, :8], old[:, :, :8]) and torch.equal(x[:, :, 72:], old[:, :, 72:])


def test_far_positions_and_positions_outside_the_table(backend, gpu_device):
    gen = torch.Generator().manual_seed(4)
    far = 131072
    table = RotaryTable(128, far, device=gpu_device)
    q, k, v = heads(gen, gpu_device, 6, torch.float32, 2, 1, 128)
    positions = torch.tensor([far - 1, 0, -1, far, 2**40, far // 2], device=gpu_device)
    kc = torch.full((2, 4, 1, 128), 7.0, device=gpu_device)
    vc = kc.clone()
    slots = torch.arange(6, dtype=torch.int32, device=gpu_device)
    out = backend.rotary_store(q, k, v, kc, vc, slots, positions, table)
    good = torch.tensor([0, 1, 5], device=gpu_device)
    check(out[good], turned(q[good], positions[good], table), "far")
    check(kc.view(8, 1, 128)[good], turned(k[good], positions[good], table), "far, stored")
    assert bool((out[2:5] == 0).all()) and bool((kc.view(8, 128)[2:5] == 7).all())
    assert bool((vc.view(8, 128)[2:5] == 7).all()) and torch.equal(vc.view(8, 1, 128)[good], v[good])


def test_non_finite_values_stay_in_their_pairs(backend, gpu_device):
    table = RotaryTable(64, 64, device=gpu_device)
    q = torch.ones(1, 1, 128, dtype=torch.bfloat16, device=gpu_device)
    q[0, 0, 3], q[0, 0, 70] = float("nan"), float("inf")
    out, _ = backend.rotary(q, q.clone(), torch.tensor([5], device=gpu_device), table)
    bad = (~torch.isfinite(out[0, 0])).nonzero().flatten().tolist()
    assert bad == [3, 35, 70]


def test_no_tokens_other_streams_and_graphs(backend, gpu_device):
    gen = torch.Generator().manual_seed(8)
    table = RotaryTable(128, 256, device=gpu_device)
    q, k, v = heads(gen, gpu_device, 40, torch.bfloat16, 8, 2, 128)
    none = backend.rotary(q[:0], k[:0], torch.empty(0, dtype=torch.int64, device=gpu_device), table)
    assert none[0].shape == (0, 8, 128)
    positions = torch.randint(0, 256, (40,), generator=gen).to(gpu_device)
    ref = backend.rotary(q, k, positions, table)
    kc = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16, device=gpu_device)
    vc = torch.zeros_like(kc)
    slots = torch.randperm(64, generator=gen)[:40].to(torch.int32).to(gpu_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = backend.rotary_store(q, k, v, kc, vc, slots, positions, table)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref[0])
    assert torch.equal(kc.view(64, 2, 128)[slots.long()], ref[1])
    # Captured: new values in the same buffers, several replays.
    q2, k2, p2 = q.clone(), k.clone(), positions.clone()
    graph = torch.cuda.CUDAGraph()
    with capture_graph(graph):
        captured = backend.rotary_store(q2, k2, v, kc, vc, slots, p2, table)
    for step in range(3):
        p2.copy_((positions + 11 * step) % 256)
        q2.copy_(q.roll(step, 0))
        graph.replay()
        torch.cuda.synchronize()
        eager = backend.rotary(q2, k2, p2, table)
        assert torch.equal(captured, eager[0])
        assert torch.equal(kc.view(64, 2, 128)[slots.long()], eager[1])


@pytest.mark.parametrize("dim,interleaved", [(128, False), (128, True), (40, True)])
@pytest.mark.parametrize("tokens", [1, 2, 33])
def test_fused_projections_are_rotated_in_place(backend, gpu_device, dim, interleaved, tokens):
    """q and k rotated where a projection left them, between its other parts:
    a row's q, k and v one after another, or head by head."""
    gen = torch.Generator().manual_seed(31)
    table = RotaryTable(dim, 64, device=gpu_device)
    fused = torch.randn(tokens, 3 * 4 * dim, generator=gen).to(torch.bfloat16).to(gpu_device)
    if interleaved:
        q, k, v = fused.view(tokens, 4, 3, dim).unbind(2)
    else:
        q, k, v = fused.view(tokens, 3, 4, dim).unbind(1)
    positions = torch.randint(0, 64, (tokens,), generator=gen).to(gpu_device)
    old_v = v.clone()
    expected = backend.rotary(q, k, positions, table)
    kc = torch.zeros(5, 16, 4, dim, dtype=torch.bfloat16, device=gpu_device)
    vc = torch.zeros_like(kc)
    slots = torch.arange(tokens, dtype=torch.int32, device=gpu_device)
    out = backend.rotary_store(q, k, v, kc, vc, slots, positions, table, q_out=q, k_out=k)
    assert out.data_ptr() == q.data_ptr()
    assert torch.equal(q, expected[0]) and torch.equal(k, expected[1]) and torch.equal(v, old_v)
    assert torch.equal(kc.view(-1, 4, dim)[:tokens], expected[1])
    assert torch.equal(vc.view(-1, 4, dim)[:tokens], old_v)
    with pytest.raises(RuntimeError, match="overlap"):
        backend.rotary(q, k, positions, table, out=(k, torch.empty_like(k)))


@pytest.mark.parametrize("sections", [(32, 0, 0), (0, 32, 0), (0, 0, 32)])
def test_one_row_of_three_positions_may_turn_every_pair(backend, gpu_device, sections):
    gen = torch.Generator().manual_seed(33)
    q, k, v = heads(gen, gpu_device, 9, torch.bfloat16, 2, 1, 64)
    positions = torch.randint(0, 50, (3, 9), generator=gen).to(gpu_device)
    got = backend.rotary(q, k, positions, RotaryTable(64, 50, sections=sections, device=gpu_device))
    plain = backend.rotary(q, k, positions[sections.index(32)].contiguous(), RotaryTable(64, 50, device=gpu_device))
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])


def test_a_cache_without_slots_stores_nothing(backend, gpu_device):
    gen = torch.Generator().manual_seed(32)
    table = RotaryTable(64, 32, device=gpu_device)
    q, k, v = heads(gen, gpu_device, 5, torch.bfloat16, 2, 1, 64)
    positions = torch.arange(5, device=gpu_device)
    kc = torch.empty(0, 16, 1, 64, dtype=torch.bfloat16, device=gpu_device)
    slots = torch.full((5,), -1, dtype=torch.int32, device=gpu_device)
    out = backend.rotary_store(q, k, v, kc, torch.empty_like(kc), slots, positions, table)
    assert torch.equal(out, backend.rotary(q, k, positions, table)[0])


def test_rows_past_4_gib(backend, gpu_device):
    table = RotaryTable(128, 16, device=gpu_device)
    nb, bs = 8400, 256  # 2 KiB rows: 4.4 GB a cache
    kc = torch.zeros(nb, bs, 8, 128, dtype=torch.bfloat16, device=gpu_device)
    vc = torch.zeros(nb, bs, 8, 128, dtype=torch.bfloat16, device=gpu_device)
    q, k, v = heads(torch.Generator().manual_seed(2), gpu_device, 3, torch.bfloat16, 8, 8, 128)
    slots = torch.tensor([nb * bs - 1, 0, nb * bs // 2], dtype=torch.int32, device=gpu_device)
    positions = torch.tensor([3, 4, 5], device=gpu_device)
    backend.rotary_store(q, k, v, kc, vc, slots, positions, table)
    ref = backend.rotary(q, k, positions, table)[1]
    rows = slots.long()
    assert torch.equal(kc.view(-1, 8, 128)[rows], ref) and torch.equal(vc.view(-1, 8, 128)[rows], v)
    assert int((kc.view(-1, 1024)[:, 0] != 0).sum()) == 3


def test_refusals(backend, gpu_device, monkeypatch):
    table = RotaryTable(128, 64, device=gpu_device)
    q, k, v = heads(torch.Generator().manual_seed(2), gpu_device, 4, torch.bfloat16, 4, 2, 128)
    positions = torch.arange(4, device=gpu_device)
    kc = torch.zeros(2, 4, 2, 128, dtype=torch.bfloat16, device=gpu_device)
    slots = torch.arange(4, dtype=torch.int32, device=gpu_device)
    for call, message in (
            (lambda: backend.rotary(q, k[:3], positions, table), "row per token"),
            (lambda: backend.rotary(q, k.float(), positions, table), "one dtype"),
            (lambda: backend.rotary(q, k, positions[:3], table), "positions"),
            (lambda: backend.rotary(q, k, positions.float(), table), "int32 or int64"),
            (lambda: backend.rotary(q, k, positions.expand(3, -1), table), "sections"),
            (lambda: backend.rotary(q[..., :64], k[..., :64], positions, table), "turns 128 dims"),
            (lambda: backend.rotary(q, k, positions.cpu(), table), "device"),
            (lambda: backend.rotary(q.transpose(1, 2), k, positions, table), "contiguous head_dim"),
            (lambda: backend.rotary(q, k, positions, table, out=(q[:2], k)), "shape"),
            (lambda: backend.rotary_store(q, k, v, kc, kc, slots[:3], positions, table), "slot_mapping"),
            (lambda: backend.rotary_store(q, k, v[:, :1], kc, kc, slots, positions, table), "matching shape")):
        with pytest.raises(ValueError, match=message):
            call()
    monkeypatch.setenv("NANOVLLM_PAGED_KV_VALIDATE_INDICES", "1")
    with pytest.raises(ValueError, match="outside"):
        backend.rotary(q, k, positions + 61, table)
