"""The checked calls on shared blocks, where a batch is refused and where it is done in spite of
a bad block: with the definitions in the extension's place, without a GPU."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sharing
from deepseekrpc_b200 import cuda_ops


class Definitions:
    """The extension's calls by the definitions, on CPU tensors."""

    @staticmethod
    def run(name, arguments, tables):
        done, moves, count, status = getattr(sharing, name)(*(t.numpy() for t in (*arguments, *tables)))
        for t, new in zip(tables, done):
            t.copy_(torch.from_numpy(new))
        return torch.from_numpy(moves), torch.tensor([count], dtype=torch.int32), torch.tensor([status], dtype=torch.int32)

    def paged_fork(self, parent, lengths, *tables):
        return self.run("paged_fork", (parent, lengths), tables)

    def paged_release(self, lengths, *tables):
        return self.run("paged_release", (lengths,), tables)

    def paged_compact(self, *tables):
        return self.run("paged_compact", (), tables)


@pytest.fixture
def ops(monkeypatch):
    monkeypatch.setattr(cuda_ops, "extension", lambda: Definitions())
    return cuda_ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def tables():
    """Rows 0 and 1 hold 100 and 70 tokens, rows 2 and 3 nothing; row 4 continues row 0."""
    held = i32([2, 2, 0, 0, 2])
    table = i32([[7, 3], [1, 9], [-1, -1], [-1, -1], [7, 8]])
    ring = i32([5, 2, 0, 4, 6, 10, 11, -1, -1, -1, -1, -1])
    shares = torch.zeros(12, dtype=torch.int32)
    shares[7] = 1
    return held, table, ring, i32([0, 7, 0, 0]), shares


LENGTHS = [100, 70, 90, 65, 100]
PARENT = [-1, -1, 0, 1, -1]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_fork_with_one_bad_parent_block_hands_out_its_moves(ops):
    t = tables()
    t[1][1, 1] = 99  # row 3's copied block; row 2 is fine
    with pytest.raises(ops.BlockError) as caught:
        ops.paged_fork(i32(PARENT), i32(LENGTHS), *t)
    moves, count = caught.value.value
    assert int(count) == 2 and t[0].tolist() == [2, 2, 2, 2, 2]
    pool = torch.arange(12 * 64)[:, None] * torch.ones(8, dtype=torch.int64)
    before = pool.clone()
    (copied,), _ = sharing.paged_copy([pool.numpy()], [], moves.numpy(), int(count))
    assert t[1][2].tolist() == [7, 5]  # the good child: its own block has its rows once they are copied
    assert np.array_equal(copied[5 * 64:5 * 64 + 26], before[3 * 64:3 * 64 + 26].numpy())


def test_whole_blocks_alone_are_told_from_a_refusal_too(ops):
    t = tables()
    t[1][0, 0] = -5
    lengths = [128, 70, 128, 0, 0]
    with pytest.raises(ops.BlockError) as caught:
        ops.paged_fork(i32([-1, -1, 0, -1, -1]), i32(lengths), *t)
    assert int(caught.value.value[1]) == 0 and t[0].tolist() == [2, 2, 2, 0, 2]


def test_a_cut_with_one_bad_block_hands_out_its_moves(ops):
    t = tables()
    t[1][1, 1] = 99  # dropped by row 1; row 4 is cut within the shared block
    with pytest.raises(ops.BlockError) as caught:
        ops.paged_release(i32([100, 10, 0, 0, 30]), *t)
    moves, count = caught.value.value
    assert int(count) == 1 and moves[0].tolist() == [7 * 64, 5 * 64, 30, 0] and t[1][4].tolist() == [5, -1]


def test_a_compaction_with_one_bad_block_hands_out_its_moves(ops):
    t = tables()
    t[1][1, 1] = 99
    with pytest.raises(ops.BlockError) as caught:
        ops.paged_compact(*t)
    moves, count = caught.value.value
    assert int(count) == len([m for m in moves.tolist() if m[2]]) == 2  # blocks 7 and 8, for 0 and 2
    assert t[1][4].tolist() == [0, 2]


def test_a_refused_batch_changes_nothing_and_says_so(ops):
    calls = [lambda t: ops.paged_fork(i32([-1, -1, 2, 1, -1]), i32(LENGTHS), *t),
             lambda t: ops.paged_release(i32([100, 70, 1, 0, 100]), *t)]
    for call in calls:
        t, before = tables(), tables()
        with pytest.raises(ops.ValidationError) as caught:
            call(t)
        assert not isinstance(caught.value, ops.BlockError) and same(t, before)
    t = tables()
    t[0][3] = 3
    before = [x.clone() for x in t]
    with pytest.raises(ops.ValidationError) as caught:
        ops.paged_compact(*t)
    assert not isinstance(caught.value, ops.BlockError) and same(t, before)


def test_good_batches_return_their_moves(ops):
    t = tables()
    moves, count = ops.paged_fork(i32(PARENT), i32(LENGTHS), *t)
    assert int(count) == 2 and moves[:2].tolist() == [[192, 320, 26, 0], [576, 128, 1, 0]]
    moves, count = ops.paged_release(i32([100, 70, 0, 0, 100]), *t)
    assert int(count) == 0
    moves, count = ops.paged_compact(*t)
    assert int(count) == 3
