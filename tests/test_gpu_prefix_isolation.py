"""What one request's cached rows may do to the others that continue its prompt: nothing.
Against the 64-bit formula, within the tolerances of the tree attention (test_gpu_tree.py)."""
from __future__ import annotations

import pytest
import torch

from test_gpu_prefix import call, problem
from test_gpu_tree import check

pytestmark = pytest.mark.gpu
VALUES = [float("nan"), float("inf"), float("-inf")]


@pytest.mark.parametrize("heads", [16, 32, 64, 128])
@pytest.mark.parametrize("prompts", [
    [(300, [(5, 1)] * 12), (64, [(9, 2)] * 3)],
    [(640, [(700, 1)] * 20)],                                # own rows of several tiles
    [(200, [(30, 3), (1, 5), (400, 2), (0, 1), (70, 8)] * 3)],  # requests across groups of 128 query rows
    [(130, [(20, 1)] * 2)],                                  # at most 64 query rows with up to 32 heads
], ids=["one node", "long", "across groups", "few rows"])
def test_non_finite_own_rows_are_their_request_s(cuda, heads, prompts):
    base, rows, masks = problem(heads, prompts, heads)
    others = [b for b in range(len(rows)) if b != 1]
    first = prompts[0][0] // 64 * 64  # of request 1's own rows
    context = int(base["context"][1])
    for i, at in enumerate((first, context - 1, context)):  # a cached row twice, then its first drafted one
        d = dict(base, pool=base["pool"].clone())
        d["pool"][rows[1][at], (slice(None), slice(5, 6), slice(34, None))[i]] = VALUES[i]
        out, status, lse = call(d, return_lse=True)
        assert int(status.item()) == 2
        check(d, rows, masks, out, lse, requests=others)


@pytest.mark.parametrize("tree", ["none", "any"])
@pytest.mark.parametrize("heads,requests", [
    (16, [(5, 3), (64, 1)]),                     # few query rows
    (16, [(0, 12), (70, 9), (128, 20)]),         # groups of 8 nodes
    (32, [(1, 7), (127, 64), (60, 10)]), (64, [(63, 5), (200, 3)]), (128, [(65, 3), (0, 2)]),
])
def test_drafted_rows_that_no_node_sees_may_hold_anything(cuda, tree, heads, requests):
    d, rows, masks = problem(heads + len(requests), [(256, requests)], heads, tree=tree)
    for b in range(len(rows)):
        n0, n1, context = int(d["cu"][b]), int(d["cu"][b + 1]), int(d["context"][b])
        seen = 0
        for word in masks[n0:n1]:
            seen |= word
        for j in range(n1 - n0):
            if tree == "any" and j % 3 == 1:  # arbitrary words leave hardly a row to nobody
                for n in range(n0, n1):
                    masks[n] &= ~(1 << j)
                seen &= ~(1 << j)
            if not seen >> j & 1:
                d["pool"][rows[b][context + j]] = VALUES[j % 3]
    d["mask"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64).cuda()
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    check(d, rows, masks, out, lse)


def test_a_drafted_row_that_one_group_sees(cuda):
    """12 nodes of 16 heads are two groups; each row is seen by one node alone."""
    d, rows, masks = problem(31, [(192, [(40, 12), (3, 12)])], 16)
    masks = [1 << (i * 5 + 3) % 12 for i in range(12)] * 2
    d["mask"] = torch.tensor(masks, dtype=torch.int64).cuda()
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    check(d, rows, masks, out, lse)


def test_more_work_than_can_be_shared_out_is_reported(cuda):
    """150 requests of 64 nodes and 128 heads whose contexts fill the longest table: more than
    2^31 units a pair of SMs.  Nothing is computed, and nothing of the 20 GB of entries is read."""
    batch, nodes, heads, stride = 150, 64, 128, (1 << 25) - 1
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.empty((batch, stride), **i32)
    d = dict(q=torch.zeros((batch * nodes, heads, 576), device="cuda", dtype=torch.bfloat16), sink=None, most=nodes,
             pool=torch.zeros((64, 576), device="cuda", dtype=torch.bfloat16), table=table,
             context=torch.full((batch,), stride * 64 - nodes, **i32), cu=torch.arange(0, batch * nodes + 1, nodes, **i32),
             mask=torch.ones(batch * nodes, device="cuda", dtype=torch.int64),
             prefix=torch.zeros(batch, **i32), holder=torch.full((batch,), -1, **i32))
    try:
        out, status, lse = call(d, return_lse=True)
        assert int(status.item()) == 1
        assert not out.any() and torch.all(torch.isneginf(lse))
    finally:
        d.clear()
        del table
        torch.cuda.empty_cache()
