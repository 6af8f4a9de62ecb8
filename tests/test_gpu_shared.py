"""Decode attention over shared prefixes on the GPU against softmax attention
of every sequence's whole context in 64 bits.

Bound per element, with u = finfo(dtype).eps / 2, ref_abs the same attention
over |V| and n keys:
  * the weights are rounded to the type (relative u each): u ref_abs in the
    weighted sum, u |ref| in the sum that divides it; the output: u |ref|;
  * fp32 sums over n keys: n 2^-24 (ref_abs + |ref|) at most;
  * scores: exact products summed over 128 dims in fp32, off by at most
    2^-17 s (s: the largest scale sum |q k|), and scaled and exponentiated
    with a few more roundings: 2^-16 s + 2^-19 relative in each weight;
  * float16 weights below 2^-14 are off by up to 2^-25 absolute, against a
    weight sum of at least 1: n 2^-25 max|v|, and 2^-25 in the output.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from nanokv.packing import capture_graph

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend(gpu_device):
    from nanokv.paged_kv import create_paged_kv_backend

    return create_paged_kv_backend("hip")


def make(device, sizes, prefixes, rests, *, kv=2, group=4, bs=16, dtype=torch.bfloat16, seed=0,
         copies=True, value=None):
    """A batch of groups: sizes[g] sequences share prefixes[g] rows; sequence
    i's context is its group's prefix and rests[i] rows more (rests[i] < 0: that
    many rows short of the prefix).  Whole blocks of a prefix are one; the
    partly filled last one is a copy (``copies``)."""
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    of = [g for g, n in enumerate(sizes) for _ in range(n)]
    ctx = [prefixes[g] + r for g, r in zip(of, rests)]
    need = [-(-c // bs) for c in ctx]
    whole = [p // bs for p in prefixes]
    total_blocks = sum(whole) + sum(need) + 7
    order = rng.sample(range(total_blocks), total_blocks)
    common = []
    for n in whole:
        common.append([order.pop() for _ in range(n)])
    width = max(1, max(need, default=1), max(whole, default=0))
    tables = torch.full((len(of), width), -1, dtype=torch.int32)
    for i, g in enumerate(of):
        row = common[g][: need[i]]
        row = row + [order.pop() for _ in range(need[i] - len(row))]
        tables[i, : len(row)] = torch.tensor(row, dtype=torch.int32)
    kc = torch.randn(total_blocks, bs, kv, 128, generator=gen).to(dtype)
    vc = torch.randn(total_blocks, bs, kv, 128, generator=gen).to(dtype)
    firsts = [sum(sizes[:g]) for g in range(len(sizes))]
    for i, g in enumerate(of):
        rows = prefixes[g] - whole[g] * bs
        if rows and i != firsts[g] and ctx[i] > whole[g] * bs:
            a, b = int(tables[firsts[g], whole[g]]), int(tables[i, whole[g]])
            if a >= 0:
                for cache in (kc, vc):
                    cache[b, :rows] = cache[a, :rows]
    q = torch.randn(len(of), kv * group + 3, 128, generator=gen).to(dtype)
    cu = torch.tensor([0] + ctx).cumsum(0).to(torch.int32)
    host = dict(q=q[:, : kv * group], kc=kc, vc=vc, tables=tables, ctx=ctx)
    dev = dict(q=q.to(device)[:, : kv * group], kc=kc.to(device), vc=vc.to(device),
               tables=tables.to(device), cu=cu.to(device),
               groups=torch.tensor([0] + sizes).cumsum(0).to(torch.int32).to(device),
               prefix=torch.tensor(prefixes, dtype=torch.int32).to(device), total=sum(ctx),
               rest=sum(c - prefixes[g] if sizes[g] > 1 and c >= prefixes[g] else c
                        for g, c in zip(of, ctx)))
    return dev, host


def reference(host, scale):
    """(attention, bound) in 64 bits."""
    dtype = host["q"].dtype
    u = torch.finfo(dtype).eps / 2
    nb, bs, kv, _ = host["kc"].shape
    out, bound = [], []
    for i, n in enumerate(host["ctx"]):
        q = host["q"][i].double()
        group = q.shape[0] // kv
        at = torch.arange(n)
        block = host["tables"][i].long()[at // bs] if n else at
        keep = (block >= 0) & (block < nb)
        rows = block[keep] * bs + (at % bs)[keep]
        if not rows.numel():
            out.append(torch.zeros_like(q))
            bound.append(torch.zeros_like(q))
            continue
        k = host["kc"].view(-1, kv, 128)[rows].double().repeat_interleave(group, 1)
        v = host["vc"].view(-1, kv, 128)[rows].double().repeat_interleave(group, 1)
        weights = (torch.einsum("hd,khd->hk", q, k) * scale).softmax(1)
        ref = torch.einsum("hk,khd->hd", weights, v)
        ref_abs = torch.einsum("hk,khd->hd", weights, v.abs())
        s = float(torch.einsum("hd,khd->hk", q.abs(), k.abs()).max()) * scale
        count = rows.numel()
        b = u * (ref_abs + 2 * ref.abs())
        b = b + (count * 2.0 ** -24 + 2 * (2.0 ** -16 * s + 2.0 ** -19)) * (ref_abs + ref.abs())
        if dtype == torch.float16:
            b = b + count * 2.0 ** -25 * float(v.abs().max()) + 2.0 ** -25
        out.append(ref)
        bound.append(b)
    return torch.stack(out), torch.stack(bound)


def check(got, host, scale, what):
    ref, bound = reference(host, scale)
    err = (got.cpu().double() - ref).abs()
    assert bool((err <= bound).all()), (
        f"{what}: {int((err > bound).sum())} off, worst {float((err - bound).max()):.3e} over")


def attend(backend, dev, scale, **kwargs):
    return backend.shared_prefix_attention_decode(
        dev["q"], dev["kc"], dev["vc"], dev["tables"], dev["cu"], dev["total"], dev["groups"],
        dev["prefix"], scale, **kwargs)


LAYOUTS = [
    # kv heads, query heads per kv head, block size, group sizes, prefixes
    (2, 8, 256, [8], [1511]),          # 64 rows: two row waves
    (8, 2, 256, [40], [700]),          # 80 rows of one tile
    (8, 2, 16, [100], [1024]),         # 200 rows: two tiles
    (4, 7, 32, [3, 1, 5, 2], [64, 100, 333, 16]),  # 21, 35 and 14 rows
    (1, 1, 16, [2, 20], [15, 17]),     # 2 and 20 rows
    (2, 16, 64, [2, 9], [257, 130]),   # 32 and 144 rows
    (3, 5, 16, [4, 4], [1, 2000]),
    (2, 4, 8, [6, 3], [90, 33]),       # blocks shorter than a chunk
    (2, 4, 24, [6, 3], [90, 241]),     # blocks that are no power of two
    (5, 3, 1000, [7], [1500]),
    (16, 1, 16, [33], [129]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv,group,bs,sizes,prefixes", LAYOUTS)
def test_matches_attention_over_the_whole_contexts(backend, gpu_device, kv, group, bs, sizes, prefixes,
                                                   dtype):
    rng = random.Random(kv * 31 + group)
    rests = [rng.choice((0, 1, 2, 15, 16, 17, 63, 64, 65, 200, 777)) for _ in range(sum(sizes))]
    dev, host = make(gpu_device, sizes, prefixes, rests, kv=kv, group=group, bs=bs, dtype=dtype,
                     seed=kv + group)
    scale = 1 / math.sqrt(128)
    out = attend(backend, dev, scale)
    check(out, host, scale, "unplanned")
    plan = backend.build_shared_prefix_plan(dev["kc"], dev["cu"], dev["total"], dev["groups"],
                                            dev["prefix"], kv * group, suffix_tokens=dev["rest"])
    buffer = torch.full_like(out, 9.0)
    assert attend(backend, dev, scale, plan=plan, out=buffer) is buffer
    check(buffer, host, scale, "planned")
    again = attend(backend, dev, scale, plan=plan)
    assert torch.equal(again, buffer), "the same call gives the same bits"


def test_no_groups_and_groups_that_share_nothing(backend, gpu_device):
    rests = [0, 1, 300, 17, 64, 129, 0, 40]
    for sizes, prefixes in (([8], [0]), ([1] * 8, [5] * 8), ([3, 0, 0, 5], [0, 7, 9, 0])):
        # (a group of one has its "prefix" in its own context)
        dev, host = make(gpu_device, sizes, prefixes, rests, seed=3)
        out = attend(backend, dev, 0.1)
        check(out, host, 0.1, str(sizes))
    dev, host = make(gpu_device, [8], [0], rests, seed=3)
    none = torch.zeros(1, dtype=torch.int32, device=gpu_device)
    out = backend.shared_prefix_attention_decode(
        dev["q"], dev["kc"], dev["vc"], dev["tables"], dev["cu"], dev["total"], none, none[:0], 0.1)
    check(out, host, 0.1, "no group")
    assert bool((out[0] == 0).all()) and bool((out[6] == 0).all()), "empty contexts give zeros"
    # Sequences in front of the first group and behind the last.
    dev, host = make(gpu_device, [2, 4, 2], [0, 100, 0], rests, seed=4)
    dev["groups"], dev["prefix"] = dev["groups"][1:3].contiguous(), dev["prefix"][1:2].contiguous()
    check(attend(backend, dev, 0.1), host, 0.1, "partly grouped")


def test_sequences_shorter_than_the_prefix_are_read_alone(backend, gpu_device):
    """Padded rows (length 0) and shorter contexts in a group; NaN in the rows
    that they do not have must not reach them."""
    rests = [5, -200, 30, -1, -120, 0, 64]
    dev, host = make(gpu_device, [7], [200], rests, seed=6)
    check(attend(backend, dev, 0.09), host, 0.09, "short ones")
    assert host["ctx"][1] == 0
    # NaN and infinities in the prefix past the short contexts' ends: the
    # sequences that see them turn NaN, the others stay as they were.
    good = attend(backend, dev, 0.09)
    block = int(host["tables"][0, 199 // 16])
    dev["kc"][block, 199 % 16] = float("nan")
    dev["vc"][block, 199 % 16] = float("inf")
    bad = attend(backend, dev, 0.09)
    for i in (1, 4):
        assert torch.equal(bad[i], good[i])
    assert bool(torch.isnan(bad[0]).all())


@pytest.mark.parametrize("rests", [[-200, 5, 30], [-1, 17, 0, 64], [-60, 8, -3, 40]])
def test_a_first_sequence_without_the_whole_prefix_shares_nothing(backend, gpu_device, rests):
    """The prefix is read through the first sequence's table: where that has
    not all of it (an empty row, a shorter context, its last blocks -1), the
    others are read through their own."""
    dev, host = make(gpu_device, [2, len(rests), 2], [70, 200, 90], [3, 9] + rests + [0, 11], seed=13)
    dev["rest"] = -1
    check(attend(backend, dev, 0.09), host, 0.09, rests)


def test_rows_outside_the_contexts_do_not_matter(backend, gpu_device):
    """NaN and infinity in every row that no context holds."""
    dev, host = make(gpu_device, [5, 3], [37, 90], [3, 0, 17, 40, 1, 2, 80, 5], bs=32, seed=7)
    good = attend(backend, dev, 0.1)
    used = torch.zeros(host["kc"].shape[:2], dtype=torch.bool)
    for i, n in enumerate(host["ctx"]):
        for t in range(n):
            used[int(host["tables"][i, t // 32]), t % 32] = True
    for cache, value in ((dev["kc"], float("nan")), (dev["vc"], float("inf"))):
        cache[~used.to(gpu_device)] = value
    assert torch.equal(attend(backend, dev, 0.1), good)


def test_bad_blocks_are_dropped(backend, gpu_device):
    for bs in (16, 24):
        dev, host = make(gpu_device, [4], [10 * bs], [3 * bs, 5, 0, 70], bs=bs, seed=8)
        for table in (host["tables"], dev["tables"]):
            table[0, 2] = -1         # in the prefix: gone for the whole group
            table[:, 4] = 10**6
            table[0, 11] = -7        # in the first one's rest
        for i in range(1, 4):
            host["tables"][i, 2] = -1
        check(attend(backend, dev, 0.1), host, 0.1, f"bs={bs}")
    dev, host = make(gpu_device, [3], [64], [9, 9, 9], seed=9)
    dev["tables"].fill_(-1)
    assert bool((attend(backend, dev, 0.1) == 0).all())


def test_large_scores_and_one_key(backend, gpu_device):
    """Scores in the hundreds: the reference max moves; one key gives v."""
    dev, host = make(gpu_device, [6], [500], [1, 2, 3, 90, 0, 7], seed=10)
    for where in (dev, host):
        where["q"] = where["q"] * 16
    check(attend(backend, dev, 0.5), host, 0.5, "large scores")
    dev, host = make(gpu_device, [4], [1], [0, 0, 0, 0], seed=11)
    out = attend(backend, dev, 0.3)
    v = host["vc"][int(host["tables"][0, 0]), 0].repeat_interleave(4, 0)
    assert torch.equal(out.cpu(), v.expand(4, -1, -1))


def test_equals_the_decode_entry_within_both_bounds(backend, gpu_device):
    dev, host = make(gpu_device, [12, 4], [900, 300], [50] * 16, kv=8, group=4, bs=256, seed=12)
    plain = backend.paged_attention_decode(dev["q"], dev["kc"], dev["vc"], dev["tables"], dev["cu"],
                                           dev["total"], 0.1)
    out = attend(backend, dev, 0.1)
    _, bound = reference(host, 0.1)
    # the decode entry's partials are fp16: 2^-11 of a head's largest sum more
    assert bool(((out - plain).cpu().double().abs() <= 2 * bound + 2.0 ** -9).all())


def test_long_contexts_and_many_groups(backend, gpu_device):
    dev, host = make(gpu_device, [5], [20000], [7000, 0, 3, 64, 1], kv=1, group=8, bs=256, seed=13)
    check(attend(backend, dev, 0.1), host, 0.1, "long")
    rng = random.Random(14)
    sizes = [rng.choice((0, 1, 2, 2, 3)) for _ in range(400)]
    prefixes = [rng.choice((0, 1, 16, 40, 100)) for _ in sizes]
    rests = [rng.randint(0, 30) for _ in range(sum(sizes))]
    dev, host = make(gpu_device, sizes, prefixes, rests, kv=2, group=2, bs=16, seed=14)
    check(attend(backend, dev, 0.1), host, 0.1, "many")


def test_understated_rest_is_served(backend, gpu_device):
    dev, host = make(gpu_device, [6], [64], [900, 5, 77, 300, 1, 2], seed=15)
    plan = backend.build_shared_prefix_plan(dev["kc"], dev["cu"], dev["total"], dev["groups"],
                                            dev["prefix"], 8, suffix_tokens=0)
    check(attend(backend, dev, 0.1, plan=plan), host, 0.1, "rest 0")


def test_graph_replays_with_new_lengths_and_groups(backend, gpu_device):
    """Plan and attention in one captured graph: the groups, prefixes and
    lengths of every replay are read from the buffers."""
    full, host_full = make(gpu_device, [6, 2], [300, 90], [200] * 8, kv=2, group=8, bs=16, seed=16)
    cu, groups, prefix = full["cu"].clone(), full["groups"].clone(), full["prefix"].clone()
    most = full["total"]

    def step():
        plan = backend.build_shared_prefix_plan(full["kc"], cu, most, groups, prefix, 16)
        return backend.shared_prefix_attention_decode(full["q"], full["kc"], full["vc"], full["tables"],
                                                      cu, most, groups, prefix, 0.1, plan=plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with capture_graph(graph):
        out = step()
    other = torch.cuda.CUDAGraph()  # a second graph beside the first
    with capture_graph(other):
        out_other = step()
    cases = [([6, 2], [300, 90], [200] * 8), ([6, 2], [32, 90], [10, 0, 299, 1, 400, 7, 60, 0]),
             ([3, 5], [0, 16], [300, 200, 5, 0, 17, 3, 16, 1]), ([8, 0], [9, 0], [0] * 8)]
    for sizes, prefixes, rests in cases:
        of = [g for g, n in enumerate(sizes) for _ in range(n)]
        ctx = [prefixes[g] + r for g, r in zip(of, rests)]
        # The rows of one sequence serve all: every table is the first one's,
        # so any prefix is shared.
        full["tables"].copy_(full["tables"][:1].expand(8, -1).clone())
        cu.copy_(torch.tensor([0] + ctx).cumsum(0).to(torch.int32))
        groups.copy_(torch.tensor([0] + sizes).cumsum(0).to(torch.int32))
        prefix.copy_(torch.tensor(prefixes, dtype=torch.int32))
        host = dict(host_full, tables=full["tables"].cpu(), ctx=ctx)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        check(out, host, 0.1, f"replay {sizes}")
        assert torch.equal(out, out_other)
        assert torch.equal(step(), out)


def test_calls_on_two_streams_at_once(backend, gpu_device):
    """Calls of different batches side by side, each with its workspace and
    with an output inside a wider row."""
    sets = []
    for seed, sizes, prefixes in ((41, [9, 3], [400, 77]), (42, [1, 20], [50, 300])):
        n = sum(sizes)
        dev, host = make(gpu_device, sizes, prefixes, [(37 * i) % 150 for i in range(n)], kv=2, group=8,
                         bs=16, seed=seed)
        plan = backend.build_shared_prefix_plan(dev["kc"], dev["cu"], dev["total"], dev["groups"],
                                                dev["prefix"], 16)
        wide = torch.full((n, 18, 128), 5.0, dtype=torch.bfloat16, device=gpu_device)
        sets.append((dev, host, plan, wide, torch.cuda.Stream()))
    for *_, stream in sets:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for dev, _, plan, wide, stream in sets:
            with torch.cuda.stream(stream):
                attend(backend, dev, 0.1, plan=plan, out=wide[:, 1:17])
    for *_, stream in sets:
        torch.cuda.current_stream().wait_stream(stream)
    for dev, host, plan, wide, _ in sets:
        check(wide[:, 1:17], host, 0.1, "side by side")
        assert torch.equal(wide[:, 1:17], attend(backend, dev, 0.1))
        assert bool((wide[:, 0] == 5).all()) and bool((wide[:, 17] == 5).all())


def test_caches_past_4_gib(backend, gpu_device):
    nb, bs = 8400, 256  # 2 KiB rows: 4.4 GB a cache
    kc = torch.zeros(nb, bs, 8, 128, dtype=torch.bfloat16, device=gpu_device)
    vc = torch.zeros(nb, bs, 8, 128, dtype=torch.bfloat16, device=gpu_device)
    gen = torch.Generator().manual_seed(17)
    used = [nb - 1, 3, nb - 2, nb // 2, 8300]
    small_k = torch.randn(len(used), bs, 8, 128, generator=gen).to(torch.bfloat16)
    small_v = torch.randn(len(used), bs, 8, 128, generator=gen).to(torch.bfloat16)
    at = torch.tensor(used, device=gpu_device)
    kc[at], vc[at] = small_k.to(gpu_device), small_v.to(gpu_device)
    local = torch.tensor([[0, 1, 2], [0, 1, 3], [0, 1, 4]], dtype=torch.int32)
    q = torch.randn(3, 16, 128, generator=gen).to(torch.bfloat16)
    ctx = [512 + 100, 512, 512 + 256]
    out = backend.shared_prefix_attention_decode(
        q.to(gpu_device), kc, vc, torch.tensor(used, dtype=torch.int32)[local.long()].to(gpu_device),
        torch.tensor([0] + ctx).cumsum(0).to(torch.int32).to(gpu_device), sum(ctx),
        torch.tensor([0, 3], dtype=torch.int32, device=gpu_device),
        torch.tensor([512], dtype=torch.int32, device=gpu_device), 0.09)
    check(out, dict(q=q, kc=small_k, vc=small_v, tables=local, ctx=ctx), 0.09, "past 4 GiB")


def test_fork_rotate_store_and_attend_together(backend, gpu_device):
    """A prompt forked three ways, its copied page, a step's rotated rows and
    the attention over the shared prefix, as one decode step runs them."""
    from nanokv.pool import DeviceBlockPool
    from nanokv.rotary import RotaryTable

    bs, kv, group, prompt = 16, 2, 4, 41
    gen = torch.Generator().manual_seed(18)
    pool = DeviceBlockPool(20, bs, max_seqs=4, max_blocks_per_seq=5, device=gpu_device)
    cache = torch.randn(2, 1, 20, bs, kv, 128, generator=gen).to(torch.bfloat16).to(gpu_device)
    table = RotaryTable(128, 64, device=gpu_device)
    pool.allocate(0, 3)
    for child in (1, 2, 3):
        pool.fork(0, child, prompt)
    pool.flush()
    backend.copy_blocks(cache, pool.copies)
    q = torch.randn(4, kv * group, 128, generator=gen).to(torch.bfloat16).to(gpu_device)
    k = torch.randn(4, kv, 128, generator=gen).to(torch.bfloat16).to(gpu_device)
    v = torch.randn(4, kv, 128, generator=gen).to(torch.bfloat16).to(gpu_device)
    tables = pool.tables[:, :3].contiguous()
    slots = (tables[:, 2] * bs + prompt % bs).to(torch.int32)
    positions = torch.full((4,), prompt, device=gpu_device)
    turned = backend.rotary_store(q, k, v, cache[0, 0], cache[1, 0], slots, positions, table)
    cu = torch.arange(5, dtype=torch.int32, device=gpu_device) * (prompt + 1)
    out = backend.shared_prefix_attention_decode(
        turned, cache[0, 0], cache[1, 0], tables, cu, 4 * (prompt + 1),
        torch.tensor([0, 4], dtype=torch.int32, device=gpu_device),
        torch.tensor([prompt], dtype=torch.int32, device=gpu_device), 0.09)
    host = dict(q=turned.cpu(), kc=cache[0, 0].cpu(), vc=cache[1, 0].cpu(), tables=tables.cpu(),
                ctx=[prompt + 1] * 4)
    check(out, host, 0.09, "step")
    assert torch.equal(cache[0, 0].view(-1, kv, 128)[slots.long()], backend.rotary(q, k, positions, table)[1])


def test_the_registered_ops_are_the_backends(backend, gpu_device):
    """torch.ops by their schemas, as a caller of the other ops finds them."""
    from nanokv.rotary import RotaryTable

    ops = torch.ops.nanovllm_paged_kv
    dev, _ = make(gpu_device, [5, 3], [130, 40], [7, 0, 33, 1, 90, 5, 5, 64], kv=2, group=4, seed=23)
    expected = attend(backend, dev, 0.1)
    plan = ops.build_shared_prefix_plan(dev["cu"], dev["groups"], dev["prefix"], 2, 8, -1)
    out = torch.empty_like(expected)
    ops.shared_prefix_attention_decode(dev["q"], dev["kc"], dev["vc"], dev["tables"], plan, 2, -1, 0.1, out)
    other = backend.build_shared_prefix_plan(dev["kc"], dev["cu"], dev["total"], dev["groups"], dev["prefix"], 8)
    other.plan, other.rest_tokens = plan, -1
    assert torch.equal(out, attend(backend, dev, 0.1, plan=other))
    table = RotaryTable(128, 300, device=gpu_device)
    positions = torch.arange(8, device=gpu_device) * 30
    q, k = dev["q"], torch.randn(8, 2, 128, device=gpu_device).to(torch.bfloat16)
    ref = backend.rotary(q, k, positions, table)
    q_out, k_out = torch.empty_like(ref[0]), torch.empty_like(ref[1])
    ops.rotary(q, k, positions, table.table, 0, [64, 64], q_out, k_out)
    assert torch.equal(q_out, ref[0]) and torch.equal(k_out, ref[1])
    kc, vc = dev["kc"].clone(), dev["vc"].clone()
    slots = torch.tensor([3, 5, -1, 7, 40, 41, 42, 43], dtype=torch.int32, device=gpu_device)
    ops.rotary_store(q, k, k, kc, vc, slots, positions, table.table, 0, [64, 64], q_out)
    backend.store(ref[1], k, dev["kc"], dev["vc"], slots)
    assert torch.equal(kc, dev["kc"]) and torch.equal(vc, dev["vc"]) and torch.equal(q_out, ref[0])
    pairs = torch.tensor([[0, 3], [1, 4]], dtype=torch.int32, device=gpu_device)
    ops.copy_blocks(kc, kc, pairs)
    backend.copy_blocks(dev["kc"], pairs)
    assert torch.equal(kc, dev["kc"]) and torch.equal(kc[3], kc[0])


def test_refusals(backend, gpu_device, monkeypatch):
    dev, _ = make(gpu_device, [4, 2], [33, 20], [5] * 6, seed=19)
    plan = backend.build_shared_prefix_plan(dev["kc"], dev["cu"], dev["total"], dev["groups"],
                                            dev["prefix"], 8)
    swap = lambda **kw: dict(dev, **kw)  # noqa: E731
    for call, message in (
            (lambda: attend(backend, dev, 0.0), "scale"),
            (lambda: attend(backend, dev, float("inf")), "scale"),
            (lambda: attend(backend, swap(q=dev["q"][:5]), 0.1), "one row per sequence"),
            (lambda: attend(backend, swap(q=dev["q"][:, :4]), 0.1, plan=plan), "built for"),
            (lambda: attend(backend, swap(groups=dev["groups"][:2]), 0.1, plan=plan), "built for"),
            (lambda: attend(backend, swap(q=dev["q"].float()), 0.1), "bfloat16 or float16"),
            (lambda: attend(backend, swap(q=dev["q"][..., :64]), 0.1), "head"),
            (lambda: attend(backend, swap(q=dev["q"].repeat(1, 5, 1)), 0.1), "query heads per kv head"),
            (lambda: attend(backend, swap(prefix=dev["prefix"][:1]), 0.1), "one entry per group"),
            (lambda: attend(backend, swap(groups=dev["groups"].long()), 0.1), "int32"),
            (lambda: attend(backend, dev, 0.1, out=dev["q"][:, :4]), "out must match"),
            (lambda: backend.build_shared_prefix_plan(dev["kc"], dev["cu"], -1, dev["groups"], dev["prefix"], 8),
             "non-negative")):
        with pytest.raises((ValueError, RuntimeError), match=message):
            call()
    # A plan of another batch under the same counts' sizes: NaN, not stale sums.
    other = make(gpu_device, [4, 2], [33, 20], [5] * 6, seed=19)[0]
    wrong = backend.build_shared_prefix_plan(dev["kc"], dev["cu"], dev["total"], dev["groups"], dev["prefix"], 8)
    wrong.plan[2] = 5
    assert bool(torch.isnan(attend(backend, other, 0.1, plan=wrong)).all())
    monkeypatch.setenv("NANOVLLM_PAGED_KV_VALIDATE_INDICES", "1")
    for groups, prefix in (([0, 4, 7], [3, 3]), ([0, 4, 3], [3, 3]), ([-1, 4, 6], [3, 3]), ([0, 4, 6], [-1, 3])):
        with pytest.raises(ValueError, match="cu_groups|prefix_lens"):
            attend(backend, swap(groups=torch.tensor(groups, dtype=torch.int32, device=gpu_device),
                                 prefix=torch.tensor(prefix, dtype=torch.int32, device=gpu_device)), 0.1)
