"""Shared blocks where something is wrong or short: what is left to the caller then."""
from __future__ import annotations

import pytest
import torch

from deepseekrpc_b200 import cuda_ops

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def tables():
    """Rows 0 and 1 hold 100 and 70 tokens, rows 2 and 3 nothing; row 4 continues row 0."""
    shares = i32([0] * 12)
    shares[7] = 1
    return (i32([2, 2, 0, 0, 2]), i32([[7, 3], [1, 9], [-1, -1], [-1, -1], [7, 8]]),
            i32([5, 2, 0, 4, 6, 10, 11, -1, -1, -1, -1, -1]), i32([0, 7, 0, 0]), shares)


def caches():
    return torch.arange(12 * 64 * 8, device="cuda").view(-1, 8), torch.zeros(12 * 64, dtype=torch.int64, device="cuda")


def test_a_fork_around_a_bad_parent_block(cuda):
    held, table, *rest = tables()
    table[1, 1] = 99  # row 3's copied block; row 2 is fine
    with pytest.raises(cuda_ops.BlockError) as caught:
        cuda_ops.paged_fork(i32([-1, -1, 0, 1, -1]), i32([100, 70, 90, 65, 100]), held, table, *rest)
    pool, generations = caches()
    before = pool.clone()
    cuda_ops.paged_copy([pool], [generations], *caught.value.value)
    assert held.tolist() == [2] * 5 and table[2].tolist() == [7, 5]
    assert torch.equal(pool[5 * 64:5 * 64 + 26], before[3 * 64:3 * 64 + 26]) and int(generations.sum()) == 26


def test_a_cut_around_a_bad_block(cuda):
    held, table, *rest = tables()
    table[1, 1] = 99  # dropped by row 1; row 4 is cut within the shared block
    with pytest.raises(cuda_ops.BlockError) as caught:
        cuda_ops.paged_release(i32([100, 10, 0, 0, 30]), held, table, *rest)
    pool, generations = caches()
    before = pool.clone()
    cuda_ops.paged_copy([pool], [generations], *caught.value.value)
    assert held.tolist() == [2, 1, 0, 0, 1] and table[4].tolist() == [5, -1]
    assert torch.equal(pool[5 * 64:5 * 64 + 30], before[7 * 64:7 * 64 + 30])


def test_a_compaction_around_a_bad_block(cuda):
    held, table, *rest = tables()
    table[1, 1] = 99
    with pytest.raises(cuda_ops.BlockError) as caught:
        cuda_ops.paged_compact(held, table, *rest)
    pool, generations = caches()
    before = pool.clone()
    cuda_ops.paged_copy([pool], [generations], *caught.value.value)
    assert table[4].tolist() == [0, 2]
    assert torch.equal(pool[:64], before[7 * 64:8 * 64]) and torch.equal(pool[2 * 64:3 * 64], before[8 * 64:9 * 64])


def test_refused_batches_are_no_block_errors(cuda):
    for call in (lambda t: cuda_ops.paged_fork(i32([-1, -1, 2, 1, -1]), i32([100, 70, 90, 65, 100]), *t),
                 lambda t: cuda_ops.paged_release(i32([100, 70, 1, 0, 100]), *t)):
        t = tables()
        with pytest.raises(cuda_ops.ValidationError) as caught:
            call(t)
        assert not isinstance(caught.value, cuda_ops.BlockError)
        for a, b in zip(t, tables()):
            assert torch.equal(a, b)
    t = tables()
    t[0][3] = 3
    with pytest.raises(cuda_ops.ValidationError) as caught:
        cuda_ops.paged_compact(*t)
    assert not isinstance(caught.value, cuda_ops.BlockError) and torch.equal(t[1], tables()[1])
