"""Decode attention over shared prefixes, on the host: what its C entry points
refuse before any launch, the sizes they lay out, and what the host binding
leaves to the backend's own checks."""
from __future__ import annotations

import pytest
import torch

from nanokv import _lib
from nanokv.paged_kv import create_paged_kv_backend

SEQS, GROUPS, KV, Q, REST = 6, 2, 2, 8, 100


def sizes(seqs=SEQS, groups=GROUPS, kv=KV, q=Q, rest=REST):
    library = _lib.load_library()
    return (library.nkv_shared_plan_bytes(seqs, groups, kv, q, rest),
            library.nkv_shared_workspace_bytes(seqs, groups, kv, q, rest))


def attend(**changes):
    """The call in order but for its pointers, which are no device's."""
    v = dict(q=4096, q_stride=Q * 128, kc=4096, vc=4096, tables=4096, width=3, plan=4096,
             plan_bytes=sizes()[0], seqs=SEQS, groups=GROUPS, kv=KV, heads=Q, dim=128, block=16, blocks=9,
             rest=REST, scale=0.1, dtype=1, workspace=4096, workspace_bytes=sizes()[1], out=4096,
             out_stride=Q * 128)
    v.update(changes)
    library = _lib.load_library()
    status = library.nkv_shared_prefix_attention_decode(
        v["q"], v["q_stride"], v["kc"], v["vc"], v["tables"], v["width"], v["plan"], v["plan_bytes"],
        v["seqs"], v["groups"], v["kv"], v["heads"], v["dim"], v["block"], v["blocks"], v["rest"],
        v["scale"], v["dtype"], v["workspace"], v["workspace_bytes"], v["out"], v["out_stride"], None)
    return status, (library.nkv_last_error() or b"").decode()


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=2), "bfloat16 and float16"), (dict(dim=64), "head_dim"), (dict(seqs=-1), "sequences"),
    (dict(seqs=_lib.NKV_MAX_PLAN_SEQS + 1), "sequences"), (dict(groups=_lib.NKV_MAX_PLAN_SEQS + 1), "sequences"), (dict(kv=3), "heads"),
    (dict(heads=34), "heads"), (dict(kv=0), "heads"), (dict(block=0), "sizes"), (dict(blocks=-1), "sizes"),
    (dict(blocks=2**28), "sizes"), (dict(width=-1), "sizes"), (dict(q_stride=Q * 128 - 8), "strides"),
    (dict(out_stride=0), "strides"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(seqs=7), "plan of"),
    (dict(groups=3), "plan of"), (dict(rest=50), "plan of"), (dict(plan_bytes=0), "plan of"),
    (dict(workspace_bytes=sizes()[1] - 1), "workspace"), (dict(q=0), "null"), (dict(kc=0), "null"),
    (dict(plan=0), "null"), (dict(workspace=0), "null"), (dict(out=0), "null"), (dict(tables=0), "null"),
    (dict(q=4096 + 8), "aligned"), (dict(plan=4096 + 8), "aligned"), (dict(q_stride=Q * 128 + 4), "aligned"),
    (dict(out=4096 + 2), "aligned"), (dict(out_stride=Q * 128 + 1), "aligned"),
])
def test_bad_calls_fail_before_launch(changes, message):
    status, error = attend(**changes)
    assert status != 0 and message in error


def test_bad_plans_fail_before_launch():
    library = _lib.load_library()

    def build(cu=4096, seqs=SEQS, groups=GROUPS, kv=KV, q=Q, rest=REST, plan=4096, nbytes=None, cu_groups=4096):
        nbytes = sizes(seqs, groups, kv, q, rest)[0] if nbytes is None else nbytes
        status = library.nkv_build_shared_plan(cu, seqs, cu_groups, 4096, groups, kv, q, rest, plan, nbytes, None)
        return status, (library.nkv_last_error() or b"").decode()

    for changes, message in ((dict(seqs=_lib.NKV_MAX_PLAN_SEQS + 1), "sequences"), (dict(kv=3), "heads"), (dict(q=64), "heads"),
                             (dict(nbytes=16), "bytes"), (dict(plan=0), "null"), (dict(cu=0), "null"),
                             (dict(cu_groups=0), "null"), (dict(plan=4096 + 4), "aligned")):
        status, error = build(**changes)
        assert status != 0 and message in error, changes


def test_sizes():
    """None for what is not supported; an unknown rest is never laid out
    smaller than a known one, nor a larger batch smaller."""
    assert sizes(seqs=_lib.NKV_MAX_PLAN_SEQS + 1) == (0, 0) and sizes(q=9) == (0, 0) and sizes(q=2 * 17) == (0, 0)
    for kv, q in ((8, 16), (1, 16), (4, 28), (4096, 4096)):
        for seqs in (1, 2, 7, 256, 4096):
            last = (0, 0)
            for rest in (0, 1, 15, 16, 1000, 10**6, 10**12, -1):
                now = sizes(seqs, max(1, seqs // 2), kv, q, rest)
                assert now[0] % 16 == 0 and now >= last
                last = now
            none = sizes(seqs, 0, kv, q, -1)
            assert 0 < none[0] <= last[0] and 0 < none[1] <= last[1]


def test_the_binding_leaves_host_tensors_to_the_general_path():
    host = _lib.load_host()
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    cache = torch.zeros((3, 16, 2, 128), dtype=torch.bfloat16)
    tables = torch.zeros((2, 1), dtype=torch.int32)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    plan = torch.zeros(4096, dtype=torch.int32)
    pairs = torch.tensor([[0, 1]], dtype=torch.int32)
    table = torch.zeros(8, 64, 2)
    positions, slots = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    assert host.shared_decode(q, cache, cache, tables, cu, 2, plan, 1, 2, 0.1, None, 0) is None
    assert host.copy_blocks(cache, cache, pairs, 0) is False
    assert host.rotary(q, q, None, None, None, None, positions, table, 0, 64, 64, None, None, 0) is None
    assert host.rotary(q, q[:, :2], q[:, :2], cache, cache, slots, positions, table, 0, 64, 64, None, None, 0) is None


def test_the_backend_refuses_host_tensors():
    backend = create_paged_kv_backend("hip")
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    cache = torch.zeros((3, 16, 2, 128), dtype=torch.bfloat16)
    tables = torch.zeros((2, 1), dtype=torch.int32)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    groups, prefix = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([1], dtype=torch.int32)
    with pytest.raises(ValueError):
        backend.build_shared_prefix_plan(cache, cu, 2, groups, prefix, 4)
    with pytest.raises(ValueError):
        backend.shared_prefix_attention_decode(q, cache, cache, tables, cu, 2, groups, prefix, 0.1)
