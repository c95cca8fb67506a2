"""Cutting requests where no block is free: first to whole blocks, which takes none and gives all
others back, then to the tokens."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sharing
from deepseekrpc_b200 import cuda_ops


def tables():
    """Three requests on the blocks 0 1 2, with 3; 4 5; 6 7 behind them; no block is free."""
    table = np.array([[0, 1, 2, 3, -1], [0, 1, 2, 4, 5], [0, 1, 2, 6, 7]], np.int32)
    return (np.array([4, 5, 5], np.int32), table, np.full(8, -1, np.int32), np.array([3, 0, 0, 0], np.int32),
            np.array([2, 2, 2, 0, 0, 0, 0, 0], np.int32))


CUTS = [  # lengths, and the copies that are left
    ([100, 300, 300], 1),  # one goes back within what it shares; its own block behind that is free by then
    ([100, 70, 0], 2),     # two within the same block, the third ends
    ([0, 0, 150], 0),      # the others end: its block is its own by then
    ([0, 0, 0], 0),
]


def whole(lengths):
    return (-(-np.asarray(lengths) // 64) * 64).astype(np.int32)


@pytest.mark.parametrize("lengths,copies", CUTS)
def test_definition(lengths, copies):
    lengths = np.array(lengths, np.int32)
    assert sharing.paged_release(lengths, *tables())[3] == int((lengths % 64 > 0).any())  # refused at once
    done, _, count, status = sharing.paged_release(whole(lengths), *tables())
    assert status == count == 0
    done, moves, count, status = sharing.paged_release(lengths, *done)
    assert status == 0 and count == copies
    held, table, ring, state, shares = done
    mapped = [table[b, j] for b in range(3) for j in range(held[b])]
    free = [ring[(state[0] + i) % 8] for i in range(state[1])]
    assert sorted({*mapped, *free}) == list(range(8)) and not set(mapped) & set(free)
    assert np.array_equal(np.bincount(mapped, minlength=8) if mapped else np.zeros(8), shares + np.isin(np.arange(8), mapped))
    sources = {int(m[0]) // 64 for m in moves[:count]}
    assert not sources & {int(m[1]) // 64 for m in moves[:count]}


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,copies", CUTS)
def test_on_the_gpu(cuda, lengths, copies):
    held, table, ring, state, shares = (torch.from_numpy(t).cuda() for t in tables())
    pool = torch.arange(8 * 64 * 8, device="cuda").view(-1, 8)
    generations = torch.zeros(8 * 64, dtype=torch.int64, device="cuda")
    rows = [pool[(table[b, :n, None] * 64 + torch.arange(64, device="cuda")).view(-1).long()].clone()
            for b, n in enumerate(held.tolist())]
    if any(n % 64 for n in lengths):
        with pytest.raises(cuda_ops.ValidationError):
            cuda_ops.paged_release(torch.tensor(lengths, dtype=torch.int32).cuda(), held, table, ring, state, shares)
    for cut in (whole(lengths), np.array(lengths, np.int32)):
        moves, count = cuda_ops.paged_release(torch.from_numpy(cut).cuda(), held, table, ring, state, shares)
        cuda_ops.paged_copy([pool], [generations], moves, count)
    assert int(count) == copies
    for b, n in enumerate(lengths):
        at = (table[b, :, None] * 64 + torch.arange(64, device="cuda")).view(-1)[:n].long()
        assert torch.equal(pool[at], rows[b][:n])
