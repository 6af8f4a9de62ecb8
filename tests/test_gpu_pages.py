"""Pages copied, forked and compacted on the GPU: bit-exact against plain
indexing and the host restatement of the block pool."""
from __future__ import annotations

import random

import pytest
import torch

from oracle.block_pool import BlockPoolOracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend(gpu_device):
    from nanokv.paged_kv import create_paged_kv_backend

    return create_paged_kv_backend("hip")


def make_pool(device, num_blocks, block_size, max_seqs, width):
    from nanokv.pool import DeviceBlockPool

    return DeviceBlockPool(num_blocks, block_size, max_seqs=max_seqs, max_blocks_per_seq=width,
                           device=device)


def assert_same(pool, oracle, what):
    snap = pool.snapshot()
    assert snap["error"] is None, (what, snap["error"])
    assert snap["queue"] == oracle.queue(), what
    assert snap["live"] == oracle.num_free() and snap["ref"] == oracle.ref, what
    assert snap["tables"] == {s: t for s, t in oracle.tables.items() if t}, what


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [
    (2, 3, 40, 16, 2, 128),  # K and V of three layers
    (37, 256, 8, 128),       # one cache, pages of many pieces
    (5, 12, 3, 1, 5),        # odd pages: 2-byte words in 16 bits
    (2, 9, 24, 1, 33),
])
def test_copy_blocks_is_bit_exact(backend, gpu_device, dtype, shape):
    gen = torch.Generator().manual_seed(sum(shape))
    cache = torch.randn(shape, generator=gen).to(dtype).to(gpu_device)
    blocks = shape[-4]
    order = torch.randperm(blocks, generator=gen).tolist()
    n = blocks // 3
    pairs = [(order[i // 2], order[blocks - 1 - i]) for i in range(n)] + [(order[0], order[0])]
    expected = cache.clone()
    flat = expected.view(-1, blocks, *shape[-3:])
    for a, b in pairs:
        flat[:, b] = flat[:, a]
    on_device = torch.tensor(pairs, dtype=torch.int32, device=gpu_device)
    for given in (pairs, on_device):
        got = cache.clone()
        backend.copy_blocks(got, given)
        assert torch.equal(got, expected)
    # Ids outside the cache, from the device, move nothing.
    outside = torch.tensor([(0, blocks), (-1, 1), (blocks, 2), (2**31 - 1, 3), (1, -5)],
                           dtype=torch.int32, device=gpu_device)
    got = cache.clone()
    backend.copy_blocks(got, outside)
    assert torch.equal(got, cache)
    # Into a cache with fewer blocks.
    small = torch.zeros(*shape[:-4], n + 1, *shape[-3:], dtype=dtype, device=gpu_device)
    backend.copy_blocks(cache, [(b, i) for i, (_, b) in enumerate(pairs[:n])], dst=small)
    for i, (_, b) in enumerate(pairs[:n]):
        assert torch.equal(small.view(-1, n + 1, *shape[-3:])[:, i], cache.view(-1, blocks, *shape[-3:])[:, b])
    backend.copy_blocks(cache, [])
    backend.copy_blocks(cache, torch.empty(0, 2, dtype=torch.int32, device=gpu_device))


def test_copy_blocks_past_4_gib_and_refusals(backend, gpu_device):
    cache = torch.zeros(2, 1100, 256, 32, 128, dtype=torch.bfloat16, device=gpu_device)  # 4.6 GB
    cache[:, 3] = torch.arange(2, device=gpu_device).to(torch.bfloat16)[:, None, None, None] + 1
    backend.copy_blocks(cache, [(3, 1099)])
    assert bool((cache[0, 1099] == 1).all()) and bool((cache[1, 1099] == 2).all())
    assert bool((cache[:, 1098] == 0).all())
    small = cache[0, :8].unsqueeze(0)
    for call, message in (
            (lambda: backend.copy_blocks(small, [(0, 8)]), "outside"),
            (lambda: backend.copy_blocks(small, [(0, 1), (2, 1)]), "twice"),
            (lambda: backend.copy_blocks(small, [(0, 1), (1, 2)]), "source"),
            (lambda: backend.copy_blocks(small, torch.zeros(3, 2, device=gpu_device)), "int32"),
            (lambda: backend.copy_blocks(small, torch.zeros(3, 3, dtype=torch.int32, device=gpu_device)), "n, 2"),
            (lambda: backend.copy_blocks(cache[:, :, :, ::2], [(0, 1)]), "contiguous"),
            (lambda: backend.copy_blocks(small[0, 0], [(0, 1)]), "caches"),
            (lambda: backend.copy_blocks(small, [(0, 1)], dst=small.float()), "number of blocks"),
            (lambda: backend.copy_blocks(small, [(0, 1)], dst=cache[:1, 4:14]), "overlap")):
        with pytest.raises(ValueError, match=message):
            call()


def test_copies_on_other_streams_and_in_graphs(backend, gpu_device):
    """Pairs read at every replay: new ones, none (-1), ids that come and go."""
    from nanokv.packing import capture_graph

    gen = torch.Generator().manual_seed(3)
    cache = torch.randn(2, 2, 12, 16, 2, 64, generator=gen).to(torch.bfloat16).to(gpu_device)
    start = cache.clone()
    pairs = torch.tensor([(0, 5), (0, 6), (1, 7)], dtype=torch.int32, device=gpu_device)

    def copied(x, of):
        x = x.clone()
        for a, b in of:
            if 0 <= a < 12 and 0 <= b < 12:
                x[:, :, b] = x[:, :, a]
        return x

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        backend.copy_blocks(cache, pairs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(cache, copied(start, pairs.tolist()))
    graph = torch.cuda.CUDAGraph()
    with capture_graph(graph):
        backend.copy_blocks(cache, pairs)
    for of in ([(5, 0), (5, 1), (6, 2)], [(-1, -1)] * 3, [(3, 8), (12, 4), (8, -2)],
               [(2, 9), (7, 10), (7, 11)]):
        pairs.copy_(torch.tensor(of, dtype=torch.int32))
        before = cache.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache, copied(before, of)), of


def test_forks_follow_the_oracle(gpu_device):
    """Random logs of allocations, appends, deallocations and forks, many
    forks in a row among them, forks of forks too."""
    rng = random.Random(5)
    bs, nb, slots, width = 16, 500, 40, 12
    pool, oracle = make_pool(gpu_device, nb, bs, slots, width), BlockPoolOracle(nb, width)
    for step in range(60):
        freed, copied_at, expected = False, {}, []
        for _ in range(rng.randint(1, 25)):
            live = [s for s in range(slots) if oracle.table(s)]
            empty = [s for s in range(slots) if not oracle.table(s)]
            kind = rng.choice(("allocate", "append", "deallocate", "fork", "fork", "fork"))
            if kind == "allocate" and empty and oracle.num_free() >= width:
                slot, n = rng.choice(empty), rng.randint(1, width - 2)
                pool.allocate(slot, n)
                oracle.allocate(slot, n)
            elif kind == "append" and live and oracle.num_free():
                slot = rng.choice(live)
                if len(oracle.table(slot)) < width:
                    pool.append(slot)
                    oracle.append(slot)
            elif kind == "deallocate" and live:
                slot = rng.choice(live)
                pool.deallocate(slot)
                oracle.deallocate(slot)
                freed = freed or bool(expected)
            elif kind == "fork" and live and empty and oracle.num_free():
                parent, child = rng.choice(live), rng.choice(empty)
                tokens = rng.randint(0, len(oracle.table(parent)) * bs)
                blocks, copied = -(-tokens // bs), tokens % bs != 0
                if copied and (freed or copied_at.get(parent) == blocks):
                    with pytest.raises(ValueError, match="flush"):
                        pool.fork(parent, child, tokens)
                    continue
                pool.fork(parent, child, tokens)
                pair = oracle.fork(parent, child, blocks, copied)
                if pair is not None:
                    expected.append(list(pair))
                    copied_at[child] = blocks
        if pool.pending_ops:
            pool.flush()
            assert pool.copies.cpu().tolist() == expected, step
        assert_same(pool, oracle, step)


def test_many_forks_of_one_prompt_in_one_log(gpu_device):
    """More children than a run of ops holds, and the queue running dry."""
    bs, children = 16, 1500
    pool = make_pool(gpu_device, 2000, bs, children + 2, 8)
    oracle = BlockPoolOracle(2000, 8)
    pool.allocate(0, 5)
    oracle.allocate(0, 5)
    expected = []
    for child in range(1, children + 1):
        pool.fork(0, child, 70)
        expected.append(list(oracle.fork(0, child, 5, True)))
    pool.flush()
    assert pool.copies.cpu().tolist() == expected
    assert_same(pool, oracle, "forked")
    assert oracle.ref[0] == children + 1
    for child in range(1, children + 1, 2):
        pool.deallocate(child)
        oracle.deallocate(child)
    pool.flush()
    assert_same(pool, oracle, "half deallocated")


def test_bad_forks_stop_the_log(gpu_device):
    """The valid prefix is applied, the first bad fork recorded, whatever
    stands behind it; the recorder's own refusals come first."""
    from nanokv import _lib

    pool = make_pool(gpu_device, 8, 4, 4, 4)

    def raw(child, blocks, parent, pair, pairs=1):
        pool._ops.append((_lib.NKV_POOL_OP_FORK, child, blocks, len(pool._args)))
        pool._args.extend((parent, pair))
        pool._pairs = pairs

    def from_parent_filled_in_the_log():
        pool.fork(0, 1, 12)
        pool.fork(1, 2, 8)  # valid: the run is cut before it

    for code, record, ok in (
            (2, lambda: raw(4, 2, 0, -1), 0), (2, lambda: raw(1, 2, -1, -1), 0),
            (2, lambda: raw(1, 2, 1, -1), 0), (3, lambda: raw(0, 1, 1, -1), 0),
            (7, lambda: raw(1, 4, 0, -1), 0), (7, lambda: raw(1, 0, 0, 0), 0),
            (7, lambda: raw(1, 3, 0, 1), 0), (7, lambda: raw(1, 3, 0, -2), 0),
            (7, lambda: pool._ops.append((_lib.NKV_POOL_OP_FORK, 1, 1, 50)), 0),
            (0, from_parent_filled_in_the_log, 2)):
        pool.reset()
        pool.allocate(0, 3)
        pool.flush()
        before = pool.snapshot()
        record()
        pool.flush()
        err, after = pool.error(), pool.snapshot()
        if code:
            assert err is not None and err[:2] == (0, code), (code, err)
            for key in ("queue", "live", "ref", "tables"):
                assert after[key] == before[key], (code, key)
        else:
            assert err is None
            assert after["tables"] == {0: [0, 1, 2], 1: [0, 1, 2], 2: [0, 1]}
            assert after["ref"][:3] == [3, 3, 2]
    # Three forks need a block each, two are free.
    pool = make_pool(gpu_device, 5, 4, 5, 4)
    pool.allocate(0, 3)
    for child in (1, 2, 3):
        pool.fork(0, child, 10)
    pool.flush()
    assert pool.error()[:2] == (3, 5)
    snap = pool.snapshot()
    assert snap["tables"] == {0: [0, 1, 2], 1: [0, 1, 3], 2: [0, 1, 4]}
    assert snap["ref"] == [3, 3, 1, 1, 1] and snap["live"] == 0
    assert pool.copies.cpu().tolist() == [[2, 3], [2, 4], [-1, -1]]
    for call in (lambda: pool.fork(0, 0, 4), lambda: pool.fork(0, 9, 4), lambda: pool.fork(0, 1, -1),
                 lambda: pool.fork(0, 1, 17)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("nb,bs,slots,width,seed", [(64, 16, 9, 8, 1), (5000, 16, 70, 60, 2),
                                                    (1, 4, 1, 1, 3), (1023, 8, 40, 30, 4)])
def test_compaction_moves_pages_and_tables(backend, gpu_device, nb, bs, slots, width, seed):
    """After compaction every sequence's context gathers to the same bytes,
    the blocks in use are the low ids, and the pool goes on as the oracle."""
    rng = random.Random(seed)
    pool, oracle = make_pool(gpu_device, nb, bs, slots, width), BlockPoolOracle(nb, width)
    gen = torch.Generator().manual_seed(seed)
    cache = torch.randn(2, 2, nb, bs, 1, 8, generator=gen).to(torch.float16).to(gpu_device)
    for turn in range(3):
        for slot in range(slots):
            n = rng.randint(1, width)
            if not oracle.table(slot) and oracle.num_free() >= n:
                shared = oracle.table(slot - 1)[: n // 2] if slot and rng.random() < 0.3 else []
                pool.allocate(slot, n, shared)
                oracle.allocate(slot, n, shared)
        for slot in range(slots):
            if rng.random() < 0.5:
                pool.deallocate(slot)
                oracle.deallocate(slot)
        held = {s: cache[:, :, torch.tensor(t, device=gpu_device)].clone()
                for s, t in oracle.tables.items() if t}
        moves = pool.compact()
        expected = oracle.compact()
        assert moves.cpu().tolist() == [list(m) for m in expected], turn
        assert_same(pool, oracle, turn)
        backend.copy_blocks(cache, moves)
        low = sum(r > 0 for r in oracle.ref)
        for s, t in oracle.tables.items():
            if t:
                assert max(t) < low
                assert torch.equal(cache[:, :, torch.tensor(t, device=gpu_device)], held[s])
    assert pool.compact().shape == (0, 2)  # nothing left to move


def test_compact_refuses_uncopied_forks(gpu_device):
    pool = make_pool(gpu_device, 16, 4, 4, 4)
    pool.allocate(0, 2)
    pool.fork(0, 1, 6)
    with pytest.raises(ValueError, match="copied"):
        pool.compact()
    pool.flush()
    assert pool.compact().shape == (0, 2)


def test_logs_with_the_launch_and_uploaded_ones_agree(gpu_device, monkeypatch):
    """The same logs at and around the length that the launch carries, and
    with none of them short enough."""
    from nanokv import _lib

    def play(slots):
        pool = make_pool(gpu_device, 3000, 16, 300, 8)
        pool.allocate(0, 3)
        for child in range(1, slots):
            pool.fork(0, child, 40)  # 4 + 2 words each
        pool.flush()
        for child in range(2, slots, 3):
            pool.deallocate(child)
        for child in range(3, slots, 3):
            pool.append(child)
        moves = pool.compact()
        return pool.snapshot(), pool.copies.tolist(), moves.tolist()

    for slots in (2, 159, 160, 161, 300):
        short = play(slots)
        with monkeypatch.context() as patch:
            patch.setattr(_lib, "NKV_POOL_LOG_WORDS", 0)
            assert play(slots) == short, slots
        assert short[0]["error"] is None


def test_copies_are_one_logs_own(gpu_device):
    """A step without calls, and a compaction, leave no pairs of an earlier
    log to be copied again."""
    pool = make_pool(gpu_device, 16, 4, 4, 4)
    pool.allocate(0, 2)
    pool.fork(0, 1, 6)
    pool.flush()
    assert pool.copies.shape == (1, 2)
    pool.flush()
    assert pool.copies.shape == (0, 2)
    pool.fork(0, 2, 5)
    pool.flush()
    pool.deallocate(1)
    assert pool.copies.shape == (1, 2)
    pool.compact()
    assert pool.copies.shape == (0, 2)


def test_a_forked_sequence_goes_on_alone(backend, gpu_device):
    """Fork, copy, store: the child's new rows reach its own page, the
    parent's stay; the shared blocks are one."""
    bs, kv = 16, 2
    pool = make_pool(gpu_device, 12, bs, 3, 6)
    cache = torch.randn(2, 1, 12, bs, kv, 128, device=gpu_device).to(torch.bfloat16)
    pool.allocate(0, 3)
    pool.fork(0, 1, 37)
    pool.fork(0, 2, 32)  # whole blocks: nothing to copy
    pool.flush()
    backend.copy_blocks(cache, pool.copies)
    tables = pool.tables.cpu()
    assert tables[1, :2].tolist() == tables[0, :2].tolist() == tables[2, :2].tolist()
    own = int(tables[1, 2])
    assert own != int(tables[0, 2]) and int(tables[2, 2]) == -1
    before = backend.gather(cache[0, 0], pool.tables[0, :3].contiguous(), 37)
    assert torch.equal(before, backend.gather(cache[0, 0], pool.tables[1, :3].contiguous(), 37))
    row = torch.randn(1, kv, 128, device=gpu_device).to(torch.bfloat16)
    slot = torch.tensor([own * bs + 37 % bs], dtype=torch.int32, device=gpu_device)
    backend.store(row, row, cache[0, 0], cache[1, 0], slot)
    child = backend.gather(cache[0, 0], pool.tables[1, :3].contiguous(), 38)
    assert torch.equal(child[:37], before) and torch.equal(child[37:], row)
    assert torch.equal(backend.gather(cache[0, 0], pool.tables[0, :3].contiguous(), 37), before)
