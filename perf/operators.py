"""Operators beside the paged KV cache: rotary positions on the way into it,
its pages copied, forked and compacted, and decode attention over a prefix
that sequences share.

Every case is one pass through one of them, on inputs made from a seed.  With
``own`` false the pass is written out in elementary torch operations, in 32
bits (64 for the angles of rotary positions); with ``own`` true it is the
calls that a serving engine makes of ``nanokv``.  ``listed()`` is the fixed
list, ``draw(rng)`` one more case of the same ranges.  A case names its kind
and sizes; sequence lengths follow from the case alone (``lengths`` seeds
them), so ``work`` knows them; values, positions and block tables follow from
the seed given to ``prepare``.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

HEAD_DIM = 128
BLOCK = 256
IMAGE_SIDE = 36  # an image span of 36 x 36 tokens
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


def listed() -> list[dict]:
    return [
        # One layer of a decode step of 64 sequences: queries and keys rotated,
        # keys and values stored. The smallest call, made once per layer.
        {"name": "rotary_decode", "kind": "rotary_store", "tokens": 64, "kv": 8, "q": 16,
         "dtype": "bf16", "rotary": 128, "layout": "half", "scaling": "none", "sections": False,
         "far": 16384},
        # One layer of a full prefill chunk of a multimodal batch: three
        # position rows (time, height, width), text and image spans.
        {"name": "rotary_chunk", "kind": "rotary_store", "tokens": 8192, "kv": 4, "q": 28,
         "dtype": "bf16", "rotary": 128, "layout": "half", "scaling": "none", "sections": True,
         "far": 32768},
        # One prompt whose keys are used where they lie (nothing is cached):
        # half of each head rotated, neighbouring pairs, a context stretched
        # eight times.
        {"name": "rotary_prompt", "kind": "rotary", "tokens": 1511, "kv": 2, "q": 16,
         "dtype": "fp16", "rotary": 64, "layout": "interleaved", "scaling": "yarn",
         "sections": False, "far": 131072},
        # Copy on write of the last page of 7 beams in one layer: latency.
        {"name": "copy_beams", "kind": "copy", "pairs": 7, "layers": 1, "kv": 2, "dtype": "bf16"},
        # Parallel sampling: one prompt with an image span admitted and forked
        # into 63 continuations, its last page copied for each in 28 layers.
        {"name": "fork_samples", "kind": "fork", "children": 63, "tokens": 1511, "layers": 28,
         "kv": 2, "dtype": "bf16"},
        # Half of 96 sequences have finished: the pages in use move to the
        # low end of the cache, 12 layers.
        {"name": "compact_half", "kind": "compact", "seqs": 96, "low": 256, "high": 8192,
         "finished": 0.5, "layers": 12, "kv": 4, "dtype": "fp16", "lengths": 9},
        # Decode attention of 8 samples of one multimodal prompt: latency.
        {"name": "shared_samples", "kind": "shared", "seqs": 8, "groups": 1, "prefix_low": 1511,
         "prefix_high": 1511, "low": 1, "high": 200, "kv": 2, "q": 16, "dtype": "bf16",
         "lengths": 4},
        # 32 questions about one long document, 7 query heads per kv head.
        {"name": "shared_document", "kind": "shared", "seqs": 32, "groups": 1, "prefix_low": 12001,
         "prefix_high": 12001, "low": 16, "high": 1024, "kv": 4, "q": 28, "dtype": "fp16",
         "lengths": 6},
        # A mixed batch: groups of unlike sizes and prefixes, sequences alone.
        {"name": "shared_groups", "kind": "shared", "seqs": 96, "groups": 13, "prefix_low": 1,
         "prefix_high": 16384, "low": 1, "high": 2048, "kv": 8, "q": 32, "dtype": "bf16",
         "lengths": 12},
        # A full decode batch behind one system prompt and its examples.
        {"name": "shared_system", "kind": "shared", "seqs": 256, "groups": 1, "prefix_low": 16384,
         "prefix_high": 16384, "low": 16, "high": 2048, "kv": 8, "q": 16, "dtype": "bf16",
         "lengths": 21},
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("rotary", "rotary_store", "rotary_store", "copy", "fork", "compact",
                       "shared", "shared", "shared"))
    kv, q = rng.choice(((8, 16), (8, 32), (4, 28), (2, 16)))
    half = rng.choice(("bf16", "bf16", "fp16"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    lengths = rng.randrange(1 << 20)
    if kind in ("rotary", "rotary_store"):
        rotary = rng.choice((128, 128, 64, 32))
        return {"kind": kind, "tokens": _log_int(rng, 1, 8192), "kv": kv, "q": q, "dtype": dtype,
                "rotary": rotary, "layout": rng.choice(("half", "half", "interleaved")),
                "scaling": rng.choice(("none", "linear", "ntk", "yarn", "bands")),
                "sections": rng.random() < 0.4, "far": _log_int(rng, 8192, 131072)}
    if kind == "copy":
        return {"kind": kind, "pairs": _log_int(rng, 1, 256), "layers": rng.choice((1, 2, 4)),
                "kv": rng.choice((2, 4)), "dtype": half}
    if kind == "fork":
        return {"kind": kind, "children": _log_int(rng, 1, 63), "tokens": _log_int(rng, 40, 4000),
                "layers": rng.choice((4, 12, 28)), "kv": 2, "dtype": half}
    if kind == "compact":
        return {"kind": kind, "seqs": _log_int(rng, 2, 96), "low": _log_int(rng, 17, 512),
                "high": _log_int(rng, 1024, 8192), "finished": round(rng.uniform(0.2, 0.8), 3),
                "layers": rng.choice((1, 4, 12)), "kv": rng.choice((2, 4)), "dtype": half,
                "lengths": lengths}
    seqs = _log_int(rng, 2, 256)
    low = _log_int(rng, 1, 16384)
    return {"kind": kind, "seqs": seqs, "groups": _log_int(rng, 1, max(1, seqs // 2)),
            "prefix_low": low, "prefix_high": _log_int(rng, low, 16384), "low": 1,
            "high": _log_int(rng, 16, 2048), "kv": kv, "q": q, "dtype": half, "lengths": lengths}


# ------------------------------------------------------------------ lengths

def _blocks(tokens: int) -> int:
    return -(-tokens // BLOCK)


def _shared_lengths(case: dict):
    """(sequences per group, prefix of each group, context of each sequence).
    A group of one sequence shares nothing: its prefix is 0."""
    rng = random.Random(int(case["lengths"]))
    groups, seqs = case["groups"], case["seqs"]
    cuts = sorted(rng.sample(range(1, seqs), groups - 1))
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [seqs])]
    prefix = [_log_int(rng, case["prefix_low"], case["prefix_high"]) if n > 1 else 0 for n in sizes]
    ctx = [p + _log_int(rng, case["low"], case["high"]) for n, p in zip(sizes, prefix) for _ in range(n)]
    return sizes, prefix, ctx


def _compact_lengths(case: dict):
    """(blocks of each sequence, whether it has finished)."""
    rng = random.Random(int(case["lengths"]))
    blocks = [_blocks(_log_int(rng, case["low"], case["high"])) for _ in range(case["seqs"])]
    done = [rng.random() < case["finished"] for _ in blocks]
    if all(done):
        done[-1] = False
    return blocks, done


def _moves(blocks, done) -> int:
    """Blocks in use at or past the number in use: each moves once."""
    used = [not d for n, d in zip(blocks, done) for _ in range(n)]
    return sum(used[sum(used):])


# ------------------------------------------------------------------- inputs

def _normal(shape, dtype, gen) -> torch.Tensor:
    return torch.randn(shape, dtype=dtype, device=DEVICE, generator=gen)


def _int32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cu(lens) -> torch.Tensor:
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _int32(out)


def _rotary_parameters(case: dict) -> dict:
    """How positions become angles, as a model's configuration says it."""
    scaling = {
        "none": None,
        "linear": {"type": "linear", "factor": 4.0},
        "ntk": {"type": "ntk", "factor": 4.0},
        "yarn": {"type": "yarn", "factor": 8.0, "original_max_position": 16384},
        "bands": {"type": "bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                  "original_max_position": 8192},
    }[case["scaling"]]
    half = case["rotary"] // 2
    sections = (half // 4, half * 3 // 8, half - half // 4 - half * 3 // 8) if case["sections"] else None
    return {"rotary_dim": case["rotary"], "max_position": case["far"], "base": 1000000.0,
            "layout": case["layout"], "scaling": scaling, "sections": sections}


def _rotary_inputs(case: dict, seed: int, gen) -> dict:
    kv, q, tokens, dtype = case["kv"], case["q"], case["tokens"], DTYPES[case["dtype"]]
    fused = _normal((tokens, (q + 2 * kv) * HEAD_DIM), dtype, gen)  # one projection's output
    parts = fused.split([q * HEAD_DIM, kv * HEAD_DIM, kv * HEAD_DIM], dim=1)
    s = dict(zip(("q", "k", "v"), (p.view(tokens, -1, HEAD_DIM) for p in parts)))
    s["rotary"] = _rotary_parameters(case)
    if case["sections"]:  # text and image spans in turn, from one start
        at = torch.arange(tokens, device=DEVICE)
        span = IMAGE_SIDE * IMAGE_SIDE
        start = torch.randint(0, max(1, case["far"] - tokens), (1,), device=DEVICE, generator=gen)
        image, inside = (at // span) % 2 == 1, at % span
        base = start + at - inside * image
        s["positions"] = torch.stack((base, base + inside // IMAGE_SIDE * image,
                                      base + inside % IMAGE_SIDE * image))
    else:
        s["positions"] = torch.randint(0, case["far"], (tokens,), device=DEVICE, generator=gen)
    if case["kind"] == "rotary_store":
        blocks = max(16, _blocks(2 * tokens))
        s["k_cache"] = _normal((blocks, BLOCK, kv, HEAD_DIM), dtype, gen)
        s["v_cache"] = _normal((blocks, BLOCK, kv, HEAD_DIM), dtype, gen)
        # A decode step's rows lie anywhere, a chunk's in runs of a block; one
        # row in 16 of a decode step is the padding of a graph's bucket.
        if tokens <= 1024:
            slots = torch.randperm(blocks * BLOCK, device=DEVICE, generator=gen)[:tokens]
            slots[15::16] = -1
        else:
            order = torch.randperm(blocks, device=DEVICE, generator=gen)
            at = torch.arange(tokens, device=DEVICE)
            slots = order[at // BLOCK] * BLOCK + at % BLOCK
        s["slots"] = slots.to(torch.int32)
    return s


def _page_inputs(case: dict, seed: int, gen) -> dict:
    s: dict = {}
    if case["kind"] == "copy":
        blocks = 3 * case["pairs"] + 5
        order = random.Random(seed).sample(range(blocks), blocks)
        # Beams fork: every second source is copied twice.
        n = case["pairs"]
        s["pairs"] = _int32([[order[i // 2 if i % 4 < 2 else n + i // 4], order[blocks - 1 - i]]
                             for i in range(n)])
    elif case["kind"] == "fork":
        s["width"] = _blocks(case["tokens"]) + 1
        blocks = s["width"] + case["children"] + 8
    else:
        per_seq, done = _compact_lengths(case)
        blocks = sum(per_seq) + 8
        s["per_seq"], s["done"] = per_seq, done
        s["width"] = max(per_seq)
        s["counts"], s["live"] = _int32(per_seq), torch.tensor([not d for d in done], device=DEVICE)
    s["blocks"] = blocks
    s["cache"] = _normal((2, case["layers"], blocks, BLOCK, case["kv"], HEAD_DIM),
                         DTYPES[case["dtype"]], gen)
    return s


def _shared_inputs(case: dict, seed: int, gen) -> dict:
    kv, q, dtype = case["kv"], case["q"], DTYPES[case["dtype"]]
    sizes, prefix, ctx = _shared_lengths(case)
    # Whole blocks of a prefix are one and the same for its group; a sequence
    # has a block of its own from the prefix's last, partly filled one on.
    shared = [p // BLOCK for p in prefix]
    rows, need = [], 0
    for g, n in enumerate(sizes):
        rows += [g] * n
    need = sum(shared) + sum(_blocks(c) - shared[g] for g, c in zip(rows, ctx))
    blocks = need + 8
    order = random.Random(seed).sample(range(blocks), blocks)
    at = 0
    common = []
    for n in shared:
        common.append(order[at: at + n])
        at += n
    width = max(_blocks(c) for c in ctx)
    tables = []
    for g, c in zip(rows, ctx):
        private = order[at: at + _blocks(c) - shared[g]]
        at += len(private)
        tables.append(common[g] + private + [-1] * (width - shared[g] - len(private)))
    s = {"tables": _int32(tables), "cu_k": _cu(ctx), "total": sum(ctx), "cu_groups": _cu(sizes),
         "prefix": _int32(prefix), "scale": HEAD_DIM ** -0.5, "most": max(sizes),
         "longest_prefix": max(prefix), "groups": len(sizes),
         "longest_rest": max(c - prefix[g] for g, c in zip(rows, ctx)),
         "rest": sum(c - prefix[g] for g, c in zip(rows, ctx))}
    s["q"] = _normal((case["seqs"], (q + 2 * kv) * HEAD_DIM), dtype, gen)[:, : q * HEAD_DIM].view(
        case["seqs"], q, HEAD_DIM)
    s["k_cache"] = _normal((blocks, BLOCK, kv, HEAD_DIM), dtype, gen)
    s["v_cache"] = _normal((blocks, BLOCK, kv, HEAD_DIM), dtype, gen)
    # The prefix's partly filled last block: every sequence's copy of it.
    firsts = s["cu_groups"][:-1].long()[torch.tensor(rows, device=DEVICE)]
    last = torch.tensor([shared[g] if prefix[g] % BLOCK else -1 for g in rows], device=DEVICE)
    here = torch.nonzero(last >= 0).flatten()
    if here.numel():
        to = s["tables"][here, last[here]].long()
        source = s["tables"][firsts[here], last[here]].long()
        for cache in (s["k_cache"], s["v_cache"]):
            filled = (prefix_rows(s["prefix"], rows, here) % BLOCK)[:, None]
            keep = (torch.arange(BLOCK, device=DEVICE)[None, :] >= filled)[:, :, None, None]
            cache[to] = torch.where(keep, cache[to], cache[source])
    return s


def prefix_rows(prefix: torch.Tensor, rows: list, here: torch.Tensor) -> torch.Tensor:
    return prefix.long()[torch.tensor(rows, device=DEVICE)][here]


def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    make = {"rotary": _rotary_inputs, "rotary_store": _rotary_inputs, "shared": _shared_inputs}
    s = make.get(case["kind"], _page_inputs)(case, int(seed), gen)
    s["case"] = dict(case)
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    if own:
        _handles(s)
    return s


def _handles(s: dict) -> None:
    """What the engine keeps: its backend, the model's rotary table, the
    block pool, the step's attention plan."""
    package = str(Path(__file__).resolve().parents[1] / "nano-vllm-multimodal_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from nanokv.paged_kv import create_paged_kv_backend

    case, kind = s["case"], s["case"]["kind"]
    backend = s["backend"] = create_paged_kv_backend("hip")
    if kind in ("rotary", "rotary_store"):
        from nanokv.rotary import RotaryTable

        s["table"] = RotaryTable(device=DEVICE, **s["rotary"])
    if kind in ("fork", "compact"):
        from nanokv.pool import DeviceBlockPool

        seqs = case["children"] + 1 if kind == "fork" else case["seqs"]
        s["pool"] = DeviceBlockPool(s["blocks"], BLOCK, max_seqs=seqs, max_blocks_per_seq=s["width"],
                                    device=DEVICE)
    if kind == "shared":
        s["plan"] = backend.build_shared_prefix_plan(
            s["k_cache"], s["cu_k"], s["total"], s["cu_groups"], s["prefix"], case["q"],
            suffix_tokens=s["rest"])


# ------------------------------------------------------- the operators' plain forms

def _inverse_frequencies(p: dict):
    """(radians per position of each pair, the factor of cosine and sine)."""
    d, base, scaling = p["rotary_dim"], p["base"], p["scaling"] or {"type": "none"}
    j = torch.arange(d // 2, dtype=torch.float64, device=DEVICE)
    kind, factor = scaling["type"], scaling.get("factor", 1.0)
    if kind == "ntk":
        base = base * factor ** (d / (d - 2))
    inv = base ** (-2.0 * j / d)
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "yarn":
        original = scaling["original_max_position"]
        low, high = (d * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
                     for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), d - 1)
        ramp = ((j - low) / max(high - low, 1e-3)).clamp(0, 1)
        return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if kind == "bands":
        original, slow, fast = (scaling[k] for k in ("original_max_position", "low_freq_factor",
                                                     "high_freq_factor"))
        smooth = ((original * inv / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        return inv * ((1 - smooth) / factor + smooth), 1.0
    return inv, 1.0


def _turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, p: dict) -> torch.Tensor:
    """x [T, H, D] in 32 bits, its first rotary_dim dims turned by the angles."""
    r = p["rotary_dim"]
    if p["layout"] == "half":
        a, b = x[..., : r // 2], x[..., r // 2: r]
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
    c, s = cos[:, None, :], sin[:, None, :]
    first, second = a * c - b * s, b * c + a * s
    turned = (torch.cat((first, second), -1) if p["layout"] == "half"
              else torch.stack((first, second), -1).flatten(-2))
    return torch.cat((turned, x[..., r:]), -1)


def _plain_rotary(s: dict):
    p = s["rotary"]
    inv, factor = _inverse_frequencies(p)
    positions = s["positions"].double()
    if p["sections"]:
        row = torch.repeat_interleave(torch.arange(3, device=DEVICE),
                                      torch.tensor(p["sections"], device=DEVICE))
        angles = positions[row].t() * inv
    else:
        angles = positions[:, None] * inv
    cos, sin = (angles.cos() * factor).float(), (angles.sin() * factor).float()
    q = _turn(s["q"].float(), cos, sin, p).to(s["q"].dtype)
    k = _turn(s["k"].float(), cos, sin, p).to(s["k"].dtype)
    if s["case"]["kind"] == "rotary":
        return q, k
    valid = s["slots"] >= 0
    to = s["slots"][valid].long()
    s["k_cache"].view(-1, *k.shape[1:])[to] = k[valid]
    s["v_cache"].view(-1, *k.shape[1:])[to] = s["v"][valid]
    return q, s["k_cache"], s["v_cache"]


def _plain_copy(s: dict):
    source, to = s["pairs"].long().unbind(1)
    s["cache"][:, :, to] = s["cache"][:, :, source]
    return s["cache"]


def _plain_fork(s: dict):
    """The prompt takes the first blocks of the free queue; a child shares
    its whole blocks and gets a fresh copy of a partly filled last one."""
    n, tokens, width = s["case"]["children"], s["case"]["tokens"], s["width"]
    need, copied = _blocks(tokens), tokens % BLOCK != 0
    queue = torch.arange(s["blocks"], dtype=torch.int32, device=DEVICE)
    tables = torch.full((n + 1, width), -1, dtype=torch.int32, device=DEVICE)
    tables[:, :need] = queue[:need]
    ref = torch.zeros(s["blocks"], dtype=torch.int32, device=DEVICE)
    ref[:need] = n + 1
    if copied:
        fresh = queue[need: need + n]
        tables[1:, need - 1] = fresh
        ref[need - 1: need + n] = 1
        s["cache"][:, :, fresh.long()] = s["cache"][:, :, need - 1: need].clone()
    return tables, ref, s["cache"]


def _plain_compact(s: dict):
    """Sequences took consecutive blocks; of U blocks in use the k-th one at
    or past U moves to the k-th free one below U."""
    counts = s["counts"].long()
    ends = counts.cumsum(0)
    columns = torch.arange(s["width"], device=DEVICE)
    ids = (ends - counts)[:, None] + columns
    held = (columns < counts[:, None]) & s["live"][:, None]
    ref = torch.zeros(s["blocks"], dtype=torch.int32, device=DEVICE)
    ref[ids[held]] = 1
    in_use = ref > 0
    low = torch.arange(s["blocks"], device=DEVICE) < in_use.sum()
    source, to = torch.nonzero(in_use & ~low).flatten(), torch.nonzero(~in_use & low).flatten()
    name = torch.arange(s["blocks"], device=DEVICE)
    name[source] = to
    tables = torch.where(held, name[ids.clamp(max=s["blocks"] - 1)], -1).to(torch.int32)
    s["cache"][:, :, to] = s["cache"][:, :, source]
    return torch.stack((source, to), 1).to(torch.int32), tables, low.to(torch.int32), s["cache"]


def _plain_shared(s: dict):
    """Scores against the prefix once per group, against the rest per
    sequence; one softmax over both."""
    case, q = s["case"], s["q"].float()
    seqs, groups, kv = case["seqs"], s["groups"], case["kv"]
    group = case["q"] // kv
    k_rows, v_rows = (s[n].view(-1, kv, HEAD_DIM) for n in ("k_cache", "v_cache"))
    cu, prefix = s["cu_groups"].long(), s["prefix"].long()
    at = torch.arange(seqs, device=DEVICE)
    of = torch.searchsorted(cu[1:].contiguous(), at, right=True)
    member = at - cu[of]
    length = (s["cu_k"][1:] - s["cu_k"][:-1]).long()
    mine = torch.minimum(prefix[of], length)
    tables = s["tables"].long().clamp(min=0)

    def rows(table, position):  # physical rows of context positions
        block = position.clamp(max=table.shape[1] * BLOCK - 1) // BLOCK
        return table.gather(1, block) * BLOCK + position % BLOCK

    # The prefix: keys [groups, kv], queries of a group padded to its most.
    p_at = torch.arange(max(1, s["longest_prefix"]), device=DEVICE)
    p_rows = rows(tables[cu[:-1]], p_at.expand(groups, -1))
    padded = torch.zeros((groups, s["most"], kv, group, HEAD_DIM), device=DEVICE)
    padded[of, member] = q.view(seqs, kv, group, HEAD_DIM)
    padded = padded.permute(0, 2, 1, 3, 4).reshape(groups * kv, -1, HEAD_DIM)
    keys = k_rows[p_rows].float().permute(0, 2, 3, 1).reshape(groups * kv, HEAD_DIM, -1)
    scores = torch.bmm(padded, keys).view(groups, kv, s["most"], group, -1)
    p_scores = scores.permute(0, 2, 1, 3, 4)[of, member] * s["scale"]  # [seqs, kv, group, P]
    p_scores = p_scores.masked_fill((p_at >= mine[:, None])[:, None, None], -math.inf)
    # The rest of each sequence.
    r_at = prefix[of][:, None] + torch.arange(max(1, s["longest_rest"]), device=DEVICE)
    r_rows = rows(tables, r_at)
    keys = k_rows[r_rows].float().permute(0, 2, 3, 1).reshape(seqs * kv, HEAD_DIM, -1)
    r_scores = torch.bmm(q.reshape(seqs * kv, group, HEAD_DIM), keys).view(seqs, kv, group, -1)
    r_scores = (r_scores * s["scale"]).masked_fill((r_at >= length[:, None])[:, None, None], -math.inf)
    # One softmax, and the products with the values.
    top = torch.maximum(p_scores.amax(-1), r_scores.amax(-1)).clamp(min=-3.0e38)[..., None]
    p_scores, r_scores = (p_scores - top).exp(), (r_scores - top).exp()
    total = p_scores.sum(-1) + r_scores.sum(-1)
    padded = torch.zeros((groups, s["most"], kv, group, p_scores.shape[-1]), device=DEVICE)
    padded[of, member] = p_scores
    padded = padded.permute(0, 2, 1, 3, 4).reshape(groups * kv, s["most"] * group, -1)
    values = v_rows[p_rows].float().permute(0, 2, 1, 3).reshape(groups * kv, -1, HEAD_DIM)
    out = torch.bmm(padded, values).view(groups, kv, s["most"], group, HEAD_DIM)
    out = out.permute(0, 2, 1, 3, 4)[of, member]
    values = v_rows[r_rows].float().permute(0, 2, 1, 3).reshape(seqs * kv, -1, HEAD_DIM)
    out = out + torch.bmm(r_scores.view(seqs * kv, group, -1), values).view(out.shape)
    out = torch.where(total[..., None] > 0, out / total[..., None], 0.0)
    return out.reshape(seqs, kv * group, HEAD_DIM).to(s["q"].dtype)


_PLAIN = {"rotary": _plain_rotary, "rotary_store": _plain_rotary, "copy": _plain_copy,
          "fork": _plain_fork, "compact": _plain_compact, "shared": _plain_shared}


def _call(s: dict):
    """The framework's calls."""
    case, backend = s["case"], s["backend"]
    kind = case["kind"]
    if kind == "rotary":
        return backend.rotary(s["q"], s["k"], s["positions"], s["table"])
    if kind == "rotary_store":
        q = backend.rotary_store(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"],
                                 s["positions"], s["table"])
        return q, s["k_cache"], s["v_cache"]
    if kind == "copy":
        backend.copy_blocks(s["cache"], s["pairs"])
        return s["cache"]
    if kind == "shared":
        return backend.shared_prefix_attention_decode(
            s["q"], s["k_cache"], s["v_cache"], s["tables"], s["cu_k"], s["total"], s["cu_groups"],
            s["prefix"], s["scale"], plan=s["plan"])
    pool = s["pool"]
    pool.reset()
    if kind == "fork":
        pool.allocate(0, _blocks(case["tokens"]))
        for child in range(1, case["children"] + 1):
            pool.fork(0, child, case["tokens"])
        pool.flush()
        backend.copy_blocks(s["cache"], pool.copies)
        return pool.tables, pool.ref, s["cache"]
    for slot, n in enumerate(s["per_seq"]):
        pool.allocate(slot, n)
    for slot, done in enumerate(s["done"]):
        if done:
            pool.deallocate(slot)
    moves = pool.compact()
    backend.copy_blocks(s["cache"], moves)
    return moves, pool.tables, pool.ref, s["cache"]


def run(s: dict):
    return _call(s) if own else _PLAIN[s["case"]["kind"]](s)


# ----------------------------------------------------------------- the rest

def work(case: dict) -> dict:
    kind = case["kind"]
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    row = case["kv"] * HEAD_DIM * size
    if kind in ("rotary", "rotary_store"):
        tokens, q_row = case["tokens"], case["q"] * HEAD_DIM * size
        angles = 8 * (3 if case["sections"] else 1) * tokens
        flops = 6 * tokens * (case["q"] + case["kv"]) * (case["rotary"] // 2)
        if kind == "rotary":
            return {"bytes": 2 * tokens * (q_row + row) + angles, "flops": flops}
        stored = tokens - (tokens // 16 if tokens <= 1024 else 0)
        return {"bytes": 2 * tokens * q_row + 4 * stored * row + 4 * tokens + angles, "flops": flops}
    page = 2 * case.get("layers", 1) * BLOCK * row
    if kind == "copy":
        n = case["pairs"]
        sources = len({i // 2 if i % 4 < 2 else n + i // 4 for i in range(n)})
        return {"bytes": (sources + n) * page + 8 * n, "flops": 0}
    if kind == "fork":
        copies = case["children"] if case["tokens"] % BLOCK else 0
        return {"bytes": (copies + (1 if copies else 0)) * page
                + 4 * (case["children"] + 1) * _blocks(case["tokens"]), "flops": 0}
    if kind == "compact":
        blocks, done = _compact_lengths(case)
        return {"bytes": _moves(blocks, done) * (2 * page + 8) + 4 * sum(blocks), "flops": 0}
    sizes, prefix, ctx = _shared_lengths(case)
    once = sum(prefix) + sum(ctx) - sum(n * p for n, p in zip(sizes, prefix))
    return {"bytes": 2 * row * once + 2 * case["seqs"] * case["q"] * HEAD_DIM * size,
            "flops": 4 * HEAD_DIM * case["q"] * sum(ctx)}


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "shared":
        return _exact_shared(s)
    if kind in ("rotary", "rotary_store"):
        return _exact_rotary(s)
    return _exact_pages(s)


def _exact_rotary(s: dict):
    p, d = s["rotary"], s["rotary"]["rotary_dim"]
    scaling = p["scaling"] or {}
    kind, f, factor = scaling.get("type"), scaling.get("factor", 1.0), 1.0
    inv = []
    for j in range(d // 2):
        w = p["base"] ** (-2 * j / d)
        if kind == "ntk":
            w = (p["base"] * f ** (d / (d - 2))) ** (-2 * j / d)
        elif kind == "linear":
            w /= f
        elif kind == "yarn":
            def dim(turns):
                return d * math.log(scaling["original_max_position"] / (turns * 2 * math.pi)) / (
                    2 * math.log(p["base"]))
            lo, hi = max(math.floor(dim(32)), 0), min(math.ceil(dim(1)), d - 1)
            share = min(1.0, max(0.0, (j - lo) / max(hi - lo, 1e-3)))
            w, factor = share * w / f + (1 - share) * w, 0.1 * math.log(f) + 1
        elif kind == "bands":
            wave = 2 * math.pi / w
            old, lo, hi = (scaling[k] for k in ("original_max_position", "low_freq_factor",
                                                "high_freq_factor"))
            if wave > old / lo:
                w /= f
            elif wave >= old / hi:
                share = (old / wave - lo) / (hi - lo)
                w = (1 - share) * w / f + share * w
        inv.append(w)
    position = s["positions"].double()
    if p["sections"]:
        which = [k for k, n in enumerate(p["sections"]) for _ in range(n)]
        angle = torch.stack([position[which[j]] * inv[j] for j in range(d // 2)], 1)
    else:
        angle = torch.stack([position * w for w in inv], 1)
    turn = torch.polar(torch.full_like(angle, factor), angle)[:, None]  # complex, [T, 1, d / 2]

    def rotate(x):
        x = x.double()
        out = x.clone()
        if p["layout"] == "half":
            z = torch.complex(x[..., : d // 2], x[..., d // 2: d]) * turn
            out[..., : d // 2], out[..., d // 2: d] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:d:2].contiguous(), x[..., 1:d:2].contiguous()) * turn
            out[..., 0:d:2], out[..., 1:d:2] = z.real, z.imag
        return out

    q, k = rotate(s["q"]), rotate(s["k"])
    if s["case"]["kind"] == "rotary":
        return q, k
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    valid = torch.nonzero(s["slots"] >= 0).flatten()
    to = s["slots"][valid].long()
    k_cache[to // BLOCK, to % BLOCK] = k[valid]
    v_cache[to // BLOCK, to % BLOCK] = s["v"][valid].double()
    return q, k_cache, v_cache


def _exact_pages(s: dict):
    """The pages one after another: their bytes are moved, never computed."""
    case, cache, kind = s["case"], s["cache"], s["case"]["kind"]
    if kind == "copy":
        moves = s["pairs"].tolist()
    elif kind == "fork":
        need = _blocks(case["tokens"])
        moves = [(need - 1, need + i) for i in range(case["children"]) if case["tokens"] % BLOCK]
    else:
        used = [not d for n, d in zip(s["per_seq"], s["done"]) for _ in range(n)]
        low = sum(used)
        holes = iter([b for b in range(low) if not used[b]])
        moves = [(b, next(holes)) for b in range(low, len(used)) if used[b]]
    for source, to in moves:  # no page is both
        cache[:, :, to] = cache[:, :, source]
    return {"copy": cache, "fork": (None, None, cache), "compact": (None, None, None, cache)}[kind]


def _exact_shared(s: dict):
    case = s["case"]
    kv, group = case["kv"], case["q"] // case["kv"]
    ends, out = s["cu_k"].tolist(), []
    for i in range(case["seqs"]):
        n = ends[i + 1] - ends[i]
        table = s["tables"][i, : _blocks(n)].long()
        k, v = (s[c][table].reshape(-1, kv, HEAD_DIM)[:n].double() for c in ("k_cache", "v_cache"))
        scores = torch.bmm(s["q"][i].double().view(kv, group, HEAD_DIM) * s["scale"],
                           k.permute(1, 2, 0).contiguous())
        out.append(torch.bmm(scores.softmax(2), v.permute(1, 0, 2).contiguous()).view(-1, HEAD_DIM))
    return torch.stack(out)
