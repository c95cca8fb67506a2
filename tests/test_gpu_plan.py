"""Block tables and slot maps built on the GPU against the definition (whole numbers: equal)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops

pytestmark = pytest.mark.gpu


def problem(seed, batch, longest, most_new, spare, shrink=False):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, longest + 1, batch).astype(np.int32)
    new = rng.integers(0, most_new + 1, batch).astype(np.int32)
    held = -(-lengths // 64)
    if shrink:  # some requests hold more than they need, some finished
        held = held + rng.integers(0, 4, batch)
        done = rng.random(batch) < 0.3
        lengths[done] = new[done] = 0
    stride = int(max(-(-(lengths + new) // 64).max(), held.max(), 1)) + 1
    need = -(-(lengths + new) // 64)
    blocks = int(held.sum() + np.maximum(need - held, 0).sum()) + spare
    ids = rng.permutation(blocks).astype(np.int32)
    table = np.full((batch, stride), -1, np.int32)
    at = 0
    for b in range(batch):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    free = ids[at:]
    ring = np.full(blocks, -7, np.int32)
    head = int(rng.integers(0, blocks))
    ring[(head + np.arange(len(free))) % blocks] = free
    state = np.array([head, len(free), 0, 0], np.int32)
    return lengths, new, held.astype(np.int32), table, ring, state


def run(args, tokens):
    """(tables, maps, cu, visible, status) of the kernel."""
    d = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in args]
    seq, pos, slots, cu, visible, status = cuda_ops.extension().paged_plan(*d, tokens)
    return [t.cpu().numpy() for t in d[2:]], [t.cpu().numpy() for t in (seq, pos, slots)], cu.cpu().numpy(), \
        visible.cpu().numpy(), int(status.item())


def check(args, tokens):
    held, table, ring, state, maps, cu, visible, status = serving.paged_plan(*args, tokens)
    got = run(args, tokens)
    assert got[4] == status
    for a, b in zip(got[0], (held, table, ring, state)):
        assert np.array_equal(a, b)
    for a, b in zip(got[1], maps):
        assert np.array_equal(a, b)
    assert np.array_equal(got[2], cu) and np.array_equal(got[3], visible)
    return got


@pytest.mark.parametrize("batch,longest,most_new", [(1, 0, 1), (1, 4096, 1), (3, 130, 200), (37, 5000, 9),
                                                    (513, 300, 3), (1025, 70, 70), (33, 0, 9000)])
@pytest.mark.parametrize("shrink", [False, True])
def test_plan_equals_the_definition(cuda, batch, longest, most_new, shrink):
    for seed in range(3):
        args = problem(seed, batch, longest, most_new, spare=seed * 5, shrink=shrink)
        pad = (0, 1, 70)[seed]  # rows behind the last token are -1
        check(args, int(args[1].sum()) + pad)


def test_plan_largest_batch(cuda):
    check(problem(5, 16384, 100, 2, spare=0), 40000)


def test_plan_no_tokens_at_all(cuda):
    check(problem(6, 4, 100, 0, spare=3), 0)


@pytest.mark.parametrize("fault", ["length", "new", "sum", "held", "held_low", "tokens", "blocks", "head", "count",
                                   "full"])
def test_refused_batch_changes_nothing(cuda, fault):
    lengths, new, held, table, ring, state = problem(7, 20, 1000, 90, spare=2, shrink=True)
    tokens = int(new.sum())
    if fault == "length":
        lengths[3] = -1
    elif fault == "new":
        new[19] = -2
    elif fault == "sum":
        lengths[0] = new[0] = 2 ** 31 - 1  # must not wrap around
    elif fault == "held":
        held[4] = table.shape[1] + 1
    elif fault == "held_low":
        held[4] = -1
    elif fault == "tokens":
        tokens -= 1
    elif fault == "blocks":
        state[1] = max(0, int(np.maximum(-(-(lengths + new) // 64) - held, 0).sum()) - 1)
    elif fault == "head":
        state[0] = len(ring)
    elif fault == "count":
        state[1] = -1
    elif fault == "full":
        state[1] = len(ring)
    got = check((lengths, new, held, table, ring, state), tokens)
    assert got[4] == 1


def test_block_ids_outside_the_pool_are_reported(cuda):
    args = list(problem(8, 6, 500, 200, spare=0))
    args[3][2, args[0][2] // 64] = len(args[4]) + 5  # the block of request 2's next token
    args[4][(args[5][0] + 1) % len(args[4])] = -3
    got = check(args, int(args[1].sum()))
    assert got[4] == 1


def test_steps_of_a_run_in_a_graph(cuda):
    """Captured once, replayed: growing, rejecting drafts, finishing; the ring turns over."""
    lengths, new, held, table, ring, state = problem(9, 8, 200, 0, spare=40)
    table = np.pad(table, ((0, 0), (0, 8)), constant_values=-1)
    new[:] = 5
    d = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (lengths, new, held, table, ring, state)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ext = cuda_ops.extension()
    ext.paged_plan(*[t.clone() for t in d], 40, status=status)  # loads the kernel before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = ext.paged_plan(*d, 40, status=status)
    expected = (lengths, new, held, table, ring, state)
    rng = np.random.default_rng(10)
    for step in range(12):
        held, table, ring, state, maps, cu, visible, code = serving.paged_plan(*expected, 40)
        graph.replay()
        assert code == 0 and int(status.item()) == 0
        for a, b in zip(d[2:], (held, table, ring, state)):
            assert np.array_equal(a.cpu().numpy(), b)
        for a, b in zip(outs, (*maps, cu, visible)):
            assert np.array_equal(a.cpu().numpy(), b)
        lengths = (lengths + rng.integers(0, 6, 8)).astype(np.int32)  # accepted drafts
        if step % 4 == 3:
            lengths[step % 8] = 0  # finished, another request starts in its place
        expected = (lengths, new, held, table, ring, state)
        d[0].copy_(torch.from_numpy(lengths))


def test_checked_call_and_refusals(cuda):
    args = [torch.from_numpy(a).cuda() for a in problem(11, 3, 100, 10, spare=1)]
    seq, pos, slots, cu, visible = cuda_ops.paged_plan(*args, 30)
    assert int(cu[-1]) == int(args[1].sum()) and visible.shape == (3,)
    args[0][0] = -5
    with pytest.raises(cuda_ops.ValidationError):
        cuda_ops.paged_plan(*args, 30)
    with pytest.raises(RuntimeError):
        cuda_ops.extension().paged_plan(args[0].long(), *args[1:], 30)
    with pytest.raises(RuntimeError):
        cuda_ops.extension().paged_plan(args[0][:2], *args[1:], 30)
    with pytest.raises(RuntimeError):
        cuda_ops.extension().paged_plan(*args[:5], args[5][:3].contiguous(), 30)
    with pytest.raises(RuntimeError):
        cuda_ops.extension().paged_plan(*args, -1)
