"""Rows of a tree attention that belong to no request: defined where the call allocates its
output, left as they are in the caller's.  Values of used rows are compared bit for bit with a
call without padding, so no tolerance enters."""
from __future__ import annotations

import math

import pytest
import torch

from deepseekrpc_b200 import _native, cuda_ops

pytestmark = pytest.mark.gpu


def problem(counts, heads, padding, dtype, context=(200, 70, 0)):
    gen = torch.Generator("cuda").manual_seed(heads + padding)
    total = sum(counts)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn((total + padding, heads, 576), generator=gen, device="cuda").to(dtype)
    q[total:] = float("nan")
    pool = torch.randn((64 * 12, 576), generator=gen, device="cuda").bfloat16()
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    return dict(q=q, pool=pool, table=torch.randperm(12, generator=gen, device="cuda").to(torch.int32).view(3, 4),
                context=i32(list(context)), cu=i32(cu), mask=torch.full((total + padding,), 7, device="cuda")), total


def call(d, total=None, most=8, **more):
    q, mask = d["q"][:total], d["mask"][:total]
    return cuda_ops.extension().tree_mla_decode(q, d["pool"], d["table"], d["context"], d["cu"], mask, most,
                                                1 / math.sqrt(192), **more)


def poison(*shapes_and_types):
    """What the allocator hands out next for these sizes holds NaN."""
    torch.cuda.synchronize()
    kept = [torch.full(shape, float("nan"), dtype=t, device="cuda") for shape, t in shapes_and_types]
    torch.cuda.synchronize()
    del kept


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts,heads,padding", [
    ((2, 0, 3), 16, 4), ((1, 1, 1), 64, 1), ((0, 0, 1), 128, 9), ((8, 8, 8), 32, 40), ((0, 0, 0), 16, 5),
])
def test_padding_rows_are_zeros(cuda, counts, heads, padding, dtype):
    d, total = problem(counts, heads, padding, dtype)
    n = total + padding
    poison(((n, heads, 512), dtype), ((n, heads), torch.float32))
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    assert torch.all(out[total:] == 0) and torch.all(torch.isneginf(lse[total:]))
    if total:
        alone = call(d, total, return_lse=True)
        assert torch.equal(out[:total], alone[0]) and torch.equal(lse[:total], alone[2])
    mine = torch.full((n, heads, 512), 7.0, dtype=dtype, device="cuda")
    poison(((n, heads), torch.float32))
    res, status, lse = call(d, out=mine, return_lse=True)
    assert int(status.item()) == 0 and torch.all(mine[total:] == 7) and torch.all(torch.isneginf(lse[total:]))
    assert torch.equal(mine[:total], out[:total])


def test_rows_of_a_refused_request_are_zeros(cuda):
    d, total = problem((2, 3, 1), 16, 2, torch.bfloat16)
    good = call(d)[0]
    d["context"][1] = -1
    poison(((8, 16, 512), torch.bfloat16))
    out, status = call(d)
    assert int(status.item()) == 1
    assert torch.all(out[2:5] == 0) and torch.all(out[6:] == 0)
    assert torch.equal(out[:2], good[:2]) and torch.equal(out[5:6], good[5:6])
    # sums in disorder: rows 0 and 1 are request 0's although request 2 starts below them
    d["context"][1] = 70
    d["cu"].copy_(torch.tensor([0, 2, 1, 8]))
    poison(((8, 16, 512), torch.bfloat16))
    out, status = call(d, most=4)  # request 2 has seven nodes
    assert int(status.item()) == 1 and torch.equal(out[:2], good[:2]) and torch.all(out[2:] == 0)


def test_replays_with_fewer_nodes(cuda):
    d, total = problem((4, 4, 4), 16, 0, torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    call(d, status=status)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(d, status=status)[0]
    for cu in ([0, 4, 8, 12], [0, 1, 1, 2], [0, 0, 0, 0], [0, 4, 4, 7]):
        d["cu"].copy_(torch.tensor(cu))
        graph.replay()
        assert int(status.item()) == 0 and torch.all(out[cu[-1]:] == 0)
        if cu[-1]:
            assert torch.equal(out[:cu[-1]], call(d, cu[-1])[0])


def test_the_c_call_leaves_or_clears_them(cuda):
    d, total = problem((1, 2, 1), 16, 3, torch.bfloat16)
    p, lib = _native.ptr, _native.library()
    size = lib.dsr_tree_mla_workspace_bytes(3, 16, 8)
    ws, err = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for flag, left in ((0, 5.0), (_native.DSR_ZERO_UNUSED, 0.0)):
        out = torch.full((7, 16, 512), 5.0, device="cuda")
        rc = lib.dsr_tree_mla_decode(p(d["q"]), _native.DSR_BF16, p(d["pool"]), 12, p(d["table"]), 4, p(d["context"]),
                                     p(d["cu"]), p(d["mask"]), 8, None, 0.07, p(out), _native.DSR_F32 | flag, None, p(ws),
                                     size, p(err), 3, 7, 16, _native.stream_handle())
        assert rc == 0 and int(err.item()) == 0
        assert torch.all(out[4:] == left) and torch.all(out[:4] != 5)
