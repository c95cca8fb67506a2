"""The plan of a batch whose requests share blocks, on the GPU against the definition: what would
reach a block of somebody else is refused, all else is as without the counts."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops
from test_gpu_sharing import problem

pytestmark = pytest.mark.gpu


def plan(lengths, new, tables, tokens, shares):
    """Runs both, and compares them; the status."""
    *four, counts = tables
    expected = serving.paged_plan(lengths, new, *four, tokens, shares=counts if shares else None)
    d = [torch.from_numpy(np.array(a, order="C")).cuda() for a in (lengths, new, *four)]
    on = torch.from_numpy(counts).cuda()
    *maps, cu, visible, status = cuda_ops.extension().paged_plan(*d, tokens, shares=on if shares else None)
    for a, b in zip((*d[2:], *maps, cu, visible), (*expected[:4], *expected[4], *expected[5:7])):
        assert np.array_equal(a.cpu().numpy(), b)
    assert int(status) == expected[7] and np.array_equal(on.cpu().numpy(), counts)
    return int(status)


@pytest.mark.parametrize("parents,children,longest", [(1, 1, 100), (1, 40, 5000), (7, 5, 64), (33, 9, 900), (600, 2, 70),
                                                      (64, 255, 200)])
def test_plan_equals_the_definition(cuda, parents, children, longest):
    for seed in range(3):
        _, lengths, tables = problem(seed, parents, children, longest, spare=2 * parents * (children + 1))
        rng = np.random.default_rng(seed + 50)
        room = tables[1].shape[1] * 64 - lengths
        new = np.minimum(rng.integers(0, 9, len(lengths)), room).astype(np.int32)
        assert plan(lengths, new, tables, int(new.sum()), True) == 0  # every request goes on behind what it has
        some = rng.random(len(lengths)) < 0.2
        cut = np.where(some, rng.integers(0, lengths + 1), lengths).astype(np.int32)
        for shares in (True, False):
            plan(cut, np.where(cut + new <= tables[1].shape[1] * 64, new, 0).astype(np.int32), tables, int(new.sum()), shares)


def two(shared_blocks, own_blocks):
    """Request 0 has a prompt of its own, request 1 the same blocks and some behind them."""
    n = shared_blocks + own_blocks
    table = np.full((2, n + 2), -1, np.int32)
    table[0, :shared_blocks] = np.arange(shared_blocks)
    table[1, :n] = np.arange(n)
    shares = np.zeros(n + 8, np.int32)
    shares[:shared_blocks] = 1
    ring = np.full(n + 8, -1, np.int32)
    ring[:8] = np.arange(n, n + 8)
    return np.array([shared_blocks, n], np.int32), table, ring, np.array([0, 8, 0, 0], np.int32), shares


@pytest.mark.parametrize("length,new,status", [
    (320, 5, 0),       # goes on
    (300, 3, 0),       # cut within its own blocks
    (192, 1, 0),       # all of its own given back but the one it writes to
    (192, 0, 0),       # none is kept beyond the prompt
    (191, 0, 0),       # cut within the last shared block: nothing is written yet
    (191, 1, 1),       # now it is
    (150, 200, 1),     # over shared blocks and into its own
    (128, 0, 1),       # a shared block would go to the ring
    (0, 0, 1), (0, 400, 1),
])
def test_a_request_that_became_shorter(cuda, length, new, status):
    lengths, fresh = np.array([192, length], np.int32), np.array([0, new], np.int32)
    assert plan(lengths, fresh, two(3, 2), new, True) == status
    assert plan(lengths, fresh, two(3, 2), new, False) == 0


def test_many_blocks_are_looked_at(cuda):
    """Every held entry counts, not the first of them alone; many CTAs, some of them ahead."""
    held, table, ring, state, shares = two(0, 20000)
    lengths = np.array([0, 0], np.int32)
    assert plan(lengths, np.zeros(2, np.int32), (held, table, ring, state, shares), 300000, True) == 0
    shares[19999] = 1
    assert plan(lengths, np.zeros(2, np.int32), (held, table, ring, state, shares), 300000, True) == 1
    shares[:] = 0
    shares[77] = 2
    assert plan(lengths, np.zeros(2, np.int32), (held, table, ring, state, shares), 300000, True) == 1
    table[1, 5] = -9  # a bad id is no shared block
    shares[77] = 0
    assert plan(lengths, np.zeros(2, np.int32), (held, table, ring, state, shares), 0, True) == 1


def test_the_checked_call(cuda):
    held, table, ring, state, shares = (torch.from_numpy(a).cuda() for a in two(3, 2))
    lengths, new = torch.tensor([192, 150], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda()
    with pytest.raises(cuda_ops.ValidationError):
        cuda_ops.paged_plan(lengths, new, held, table, ring, state, 1, shares=shares)
    assert held.tolist() == [3, 5] and table[1].tolist() == [0, 1, 2, 3, 4, -1, -1] and int(state[1]) == 8
    pool, generations = torch.zeros((len(ring) * 64, 8), device="cuda"), torch.zeros(len(ring) * 64, dtype=torch.int64).cuda()
    cuda_ops.paged_copy([pool], [generations], *cuda_ops.paged_release(lengths, held, table, ring, state, shares))
    seq, positions, slots, _, _ = cuda_ops.paged_plan(lengths, new, held, table, ring, state, 1, shares=shares)
    assert positions.tolist() == [150] and int(slots) // 64 == int(table[1, 2]) == 5  # a block of its own
    for bad in (shares[:3], shares.long(), shares.cpu()):
        with pytest.raises(RuntimeError):
            cuda_ops.paged_plan(lengths, new, held, table, ring, state, 1, shares=bad)
