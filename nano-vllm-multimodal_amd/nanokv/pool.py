"""Device block pool: the block bookkeeping of the reference BlockManager
(free-block FIFO, reference counts, per-sequence block tables;
nanovllm/engine/block_manager.py:87-118, 185-236) resident in HBM.

The scheduler keeps making its decisions as the reference does; every
BlockManager call it makes is recorded here, in the same order, and
`flush()` replays the log on the device in one launch (nkv_pool_apply).  The
device tables then feed the packers directly
(DevicePacker.pack_decode_pool / pack_prefill_pool), so per step only the op
log (a few ints per call) travels to the device, never the block lists.  The
prefix-hash chain stays with the caller, which passes each allocation's
cached-prefix block ids.
"""
from __future__ import annotations

import ctypes
from array import array
from contextlib import nullcontext
from itertools import chain
from typing import Iterable

import numpy as np
import torch

from nanokv import _lib
from nanokv.paged_kv.ops import current_stream_handle, is_current_device

_HERE = nullcontext()


class DeviceBlockPool:
    """`num_blocks` blocks of `block_size` tokens, block tables for
    `max_seqs` sequence slots of up to `max_blocks_per_seq` blocks.  The
    state lives in one device buffer owned by this object."""

    def __init__(self, num_blocks: int, block_size: int, *, max_seqs: int,
                 max_blocks_per_seq: int, device: torch.device | str) -> None:
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("DeviceBlockPool requires a ROCm (cuda) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if block_size <= 0:
            raise ValueError("block_size must be positive")
        lib = _lib.load_library()
        nbytes = int(lib.nkv_pool_bytes(num_blocks, max_seqs, max_blocks_per_seq))
        if nbytes <= 0:
            raise ValueError(
                "need 0 < num_blocks, 0 < max_seqs and 0 < max_blocks_per_seq <= num_blocks "
                "(within the library's limits)"
            )
        self.num_blocks = int(num_blocks)
        self.block_size = int(block_size)
        self.max_seqs = int(max_seqs)
        self.width = int(max_blocks_per_seq)
        self.memory = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        offsets = (ctypes.c_int64 * 6)()
        _lib.check(lib.nkv_pool_offsets(num_blocks, max_seqs, max_blocks_per_seq, offsets),
                   "nkv_pool_offsets")
        o = list(offsets)
        nb, s, w = self.num_blocks, self.max_seqs, self.width
        self.meta = self.memory[o[0]:o[0] + 64].view(torch.int64)
        self.ring = self.memory[o[1]:o[1] + 8 * nb].view(torch.int32)
        self.qpos = self.memory[o[2]:o[2] + 8 * nb].view(torch.int64)
        self.ref = self.memory[o[3]:o[3] + 4 * nb].view(torch.int32)
        self.tables = self.memory[o[4]:o[4] + 4 * s * w].view(torch.int32).view(s, w)
        self.nblk = self.memory[o[5]:o[5] + 4 * s].view(torch.int32)
        self._desc = _lib.PoolDesc(self.memory.data_ptr(), nb, s, w)
        self._ops: list[tuple[int, int, int, int]] = []
        self._args: list[int] = []
        self._run: set[int] = set()
        self._pairs = 0  # pages that the log's forks copy
        self._freed = False  # whether a deallocation follows the log's first copying fork
        self._copied: dict[int, int] = {}  # children of the log's copying forks: their block counts
        self.copies = torch.empty((0, 2), dtype=torch.int32, device=self.device)
        self._staging: torch.Tensor | None = None
        self._uploaded: torch.cuda.Event | None = None
        self.reset()

    # -------------------------------------------------------------- control
    def _stream(self) -> int:
        return current_stream_handle(self.device)

    def _on_device(self):
        """The default stream's handle is 0 on every GPU: a launch on it
        runs on the current one."""
        return _HERE if is_current_device(self.device.index) else torch.cuda.device(self.device)

    @property
    def desc(self) -> _lib.PoolDesc:
        return self._desc

    def reset(self) -> None:
        """Every block free in id order, every table empty, no error; drops
        the unflushed log."""
        self._ops.clear()
        self._args.clear()
        self._run.clear()
        self._pairs, self._freed = 0, False
        self._copied.clear()
        self.copies = self.copies[:0]
        with self._on_device():
            status = _lib.load_library().nkv_pool_init(ctypes.byref(self._desc), self._stream())
        _lib.check(status, "nkv_pool_init")

    def _check_slot(self, slot: int) -> int:
        slot = int(slot)
        if not 0 <= slot < self.max_seqs:
            raise ValueError(f"slot {slot} outside [0, {self.max_seqs})")
        return slot

    # ---------------------------------------------- the BlockManager calls
    def allocate(self, slot: int, num_blocks: int, cached: Iterable[int] = ()) -> None:
        """BlockManager.allocate (block_manager.py:185-214) for the sequence
        in `slot`, whose `num_blocks` blocks start with the cached-prefix
        ids that can_allocate found."""
        slot = self._check_slot(slot)
        cached = [int(b) for b in cached]
        if not 0 <= len(cached) <= num_blocks <= self.width:
            raise ValueError("need len(cached) <= num_blocks <= max_blocks_per_seq")
        if len(set(cached)) != len(cached) or any(not 0 <= b < self.num_blocks for b in cached):
            raise ValueError("cached block ids must be distinct and inside the pool")
        self._run.clear()
        self._ops.append((_lib.NKV_POOL_OP_ALLOCATE, slot, int(num_blocks), len(self._args)))
        self._args.append(len(cached))
        self._args.extend(cached)

    def deallocate(self, slot: int) -> None:
        """BlockManager.deallocate (block_manager.py:216-227)."""
        slot = self._check_slot(slot)
        self._run.clear()
        self._freed = self._freed or self._pairs > 0
        self._ops.append((_lib.NKV_POOL_OP_DEALLOCATE, slot, 0, 0))

    def append(self, slot: int) -> None:
        """One more block for `slot` (BlockManager.may_append when it
        allocates)."""
        slot = self._check_slot(slot)
        if slot in self._run:  # a run of appends must name distinct slots
            self._ops.append((_lib.NKV_POOL_OP_FENCE, 0, 0, 0))
            self._run.clear()
        self._run.add(slot)
        self._ops.append((_lib.NKV_POOL_OP_APPEND, slot, 0, 0))

    def may_append(self, slot: int, seq_len: int) -> bool:
        """block_manager.py:233-236: a new block when the sequence's next
        token opens one (len(seq) % block_size == 1)."""
        if int(seq_len) % self.block_size == 1:
            self.append(slot)
            return True
        return False

    # ------------------------------------- what BlockManager does not have
    def fork(self, parent: int, child: int, num_tokens: int) -> None:
        """`child` (empty) continues `parent`'s first `num_tokens` tokens:
        their whole blocks are held once more, a partly filled last one is
        replaced by a fresh block from the queue front, whose page has to be
        copied: after flush(), `copies` lists these {source, destination}
        pairs in the order of the forks
        (``backend.copy_blocks(cache, pool.copies)``)."""
        parent, child = self._check_slot(parent), self._check_slot(child)
        num_tokens = int(num_tokens)
        if parent == child:
            raise ValueError("a sequence cannot be forked into its own slot")
        blocks = -(-num_tokens // self.block_size)
        if num_tokens < 0 or blocks > self.width:
            raise ValueError("need 0 <= num_tokens <= max_blocks_per_seq blocks of tokens")
        copied = num_tokens % self.block_size != 0
        if copied and self._freed:
            raise ValueError("the log frees blocks after a fork: flush and copy that fork's pages "
                             "first, a freed source could become this fork's destination")
        if copied and self._copied.get(parent) == blocks:
            raise ValueError("the log forks a fork at its copied page: fork its parent, or flush and "
                             "copy the pages first")
        if copied:
            self._copied[child] = blocks
        self._run.clear()
        self._ops.append((_lib.NKV_POOL_OP_FORK, child, blocks, len(self._args)))
        self._args.extend((parent, self._pairs if copied else -1))
        self._pairs += 1 if copied else 0

    def compact(self) -> torch.Tensor:
        """Applies the log, then moves the blocks in use to the low ids: of U
        of them, the k-th at or past U to the k-th free one below.  Tables
        and reference counts follow, the free queue becomes U, U + 1, ...
        Returns the moves as [n, 2] int32 pairs {old, new} on the device,
        for ``backend.copy_blocks(cache, moves)`` and for the caller's own
        block ids (its prefix hashes).  Reads their number back (one
        synchronisation).  Pages that earlier forks copy must have been
        copied: with any in the log, flush and copy first."""
        if self._pairs:
            raise ValueError("the log holds forks whose pages are not copied: flush and copy them first")
        self._run.clear()
        self._ops.append((_lib.NKV_POOL_OP_COMPACT, 0, 0, len(self._args)))
        self._args.append(0)
        moves = torch.empty((max(1, self.num_blocks // 2), 2), dtype=torch.int32, device=self.device)
        self._flush(moves)
        self.copies = self.copies[:0]  # an earlier flush's: their ids have moved
        meta = self.meta.cpu().tolist()
        if meta[4]:
            raise RuntimeError(f"block pool op {int(meta[3]) - 1} failed: "
                               f"{_lib.NKV_POOL_ERRORS.get(int(meta[4]), '?')} (code {int(meta[4])})")
        return moves[: int(meta[5])]

    @property
    def pending_ops(self) -> int:
        return len(self._ops)

    def flush(self, timer=None) -> None:
        """Replay the recorded calls on the device (current stream), in
        order, and start a new log.  A short log goes with the launch; a
        longer one through a pinned staging buffer that is reused once the
        previous upload has completed.  `timer` (a
        nanokv.benchmark.LaunchTimer) brackets the apply kernel alone."""
        if not self._ops:
            self.copies = self.copies[:0]  # the last log's are not copied twice
            return
        copies = torch.empty((self._pairs, 2), dtype=torch.int32, device=self.device)
        self._flush(copies, timer)
        self.copies = copies

    def _flush(self, copies: torch.Tensor, timer=None) -> None:
        # A log that the launch can carry needs no upload (reset, one sequence
        # forked three times, its pages copied: 34.0 us with it, 20.6 without).
        with self._on_device():
            if 4 * len(self._ops) + len(self._args) <= _lib.NKV_POOL_LOG_WORDS:
                self._flush_small(copies, timer)
            else:
                self._flush_large(copies, timer)
        self._ops.clear()
        self._args.clear()
        self._run.clear()
        self._pairs, self._freed = 0, False
        self._copied.clear()

    def _flush_small(self, copies: torch.Tensor, timer) -> None:
        """A log that goes with the launch itself."""
        log = array("i", chain.from_iterable(self._ops))
        log.extend(self._args)
        at, _ = log.buffer_info()
        started = timer.start() if timer is not None else None
        status = _lib.load_library().nkv_pool_apply_log(
            ctypes.byref(self._desc), at, len(self._ops), at + 16 * len(self._ops), len(self._args),
            copies.data_ptr() if copies.numel() else None, copies.shape[0], self._stream(),
        )
        if timer is not None:
            timer.stop(started)
        _lib.check(status, "nkv_pool_apply")

    def _flush_large(self, copies: torch.Tensor, timer) -> None:
        """A log that is uploaded first."""
        ops = np.asarray(self._ops, dtype=np.int32).reshape(-1)
        args = np.asarray(self._args, dtype=np.int32)
        total = ops.size + max(args.size, 1)
        if self._uploaded is not None:
            self._uploaded.synchronize()
        if self._staging is None or self._staging.numel() < total:
            self._staging = torch.empty(max(total, 4096), dtype=torch.int32, pin_memory=True)
        host = self._staging.numpy()
        host[: ops.size] = ops
        host[ops.size: ops.size + args.size] = args
        device_log = torch.empty(total, dtype=torch.int32, device=self.device)
        device_log.copy_(self._staging[:total], non_blocking=True)
        if self._uploaded is None:
            self._uploaded = torch.cuda.Event()
        self._uploaded.record(torch.cuda.current_stream(self.device))
        started = timer.start() if timer is not None else None
        status = _lib.load_library().nkv_pool_apply_copies(
            ctypes.byref(self._desc), device_log.data_ptr(), len(self._ops),
            device_log[ops.size:].data_ptr(), args.size,
            copies.data_ptr() if copies.numel() else None, copies.shape[0], self._stream(),
        )
        if timer is not None:
            timer.stop(started)
        _lib.check(status, "nkv_pool_apply")

    # ---------------------------------------------------------------- reads
    def error(self) -> tuple[int, int, str] | None:
        """(op index, code, meaning) of the first failed op of the logs
        applied so far, or None.  Synchronizes the stream."""
        meta = self.meta.cpu().tolist()
        if meta[4] == 0:
            return None
        return int(meta[3]) - 1, int(meta[4]), _lib.NKV_POOL_ERRORS.get(int(meta[4]), "?")

    def check(self) -> None:
        err = self.error()
        if err is not None:
            raise RuntimeError(f"block pool op {err[0]} failed: {err[2]} (code {err[1]})")

    def snapshot(self) -> dict:
        """Host copy of the state (synchronizes): the free queue in order,
        the reference counts and every non-empty table."""
        meta = self.meta.cpu().tolist()
        head, tail, live = meta[0], meta[1], meta[2]
        ring = self.ring.cpu().numpy()
        cap = ring.size
        positions = np.arange(head, tail, dtype=np.int64) % cap
        queue = [int(b) for b in ring[positions] if b >= 0]
        nblk = self.nblk.cpu().numpy()
        tables = self.tables.cpu().numpy()
        return {
            "queue": queue,
            "live": int(live),
            "ref": self.ref.cpu().tolist(),
            "tables": {s: tables[s, : nblk[s]].tolist() for s in range(self.max_seqs) if nblk[s] > 0},
            "error": None if meta[4] == 0 else (int(meta[3]) - 1, int(meta[4])),
        }
