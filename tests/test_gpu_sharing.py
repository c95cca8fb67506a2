"""Forking, cutting and compacting requests, and the copies they name, on the GPU against
the definitions (whole numbers and copied bits: equal)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sharing
from deepseekrpc_b200 import cuda_ops

pytestmark = pytest.mark.gpu


def gpu(arrays):
    return [torch.from_numpy(np.array(a, order="C")).cuda() for a in arrays]


def problem(seed, parents, children, longest, spare=4, fork=False):
    """Parents, then children on their blocks (or, to be forked, without any)."""
    rng = np.random.default_rng(seed)
    n = parents * children
    lengths = rng.integers(0, longest + 1, parents)
    source = rng.integers(0, parents, n)
    cut = rng.integers(0, lengths[source] + 1)
    held = -(-lengths // 64)
    stride = int(held.max(initial=1)) + 2
    grown = np.minimum(cut + rng.integers(0, 130, n), stride * 64) if not fork else cut
    private = -(-grown // 64) - cut // 64
    blocks = int(held.sum() + private.sum()) + parents + n + spare
    ids = rng.permutation(blocks).astype(np.int32)
    table = np.full((parents + n, stride), -1, np.int32)
    at = 0
    for b in range(parents):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    for i in range(n if not fork else 0):
        b, whole = parents + i, cut[i] // 64
        table[b, :whole] = table[source[i], :whole]
        table[b, whole:whole + private[i]] = ids[at:at + private[i]]
        at += private[i]
    free = ids[at:]
    ring = np.full(blocks, -7, np.int32)
    head = int(rng.integers(0, blocks))
    ring[(head + np.arange(len(free))) % blocks] = free
    mapped = np.zeros(blocks, np.int64)
    np.add.at(mapped, table[table >= 0], 1)
    total = np.concatenate([lengths, grown]).astype(np.int32)
    parent = np.concatenate([np.full(parents, -1), np.where(rng.random(n) < 0.9, source, -1)]).astype(np.int32)
    full = np.concatenate([held, np.zeros(n, np.int64) if fork else -(-grown // 64)]).astype(np.int32)
    order = rng.permutation(parents + n)  # rows in any order
    where = np.argsort(order)
    parent = np.where(parent >= 0, where[parent], -1)[order].astype(np.int32)
    if fork:  # rows that are not forked hold nothing and have no tokens
        total = np.where((np.arange(parents + n) >= parents)[order] & (parent < 0), 0, total[order]).astype(np.int32)
    else:
        total = total[order]
    tables = (full[order], table[order], ring, np.array([head, len(free), 0, 0], np.int32),
              np.maximum(mapped - 1, 0).astype(np.int32))
    return parent, total, tables


def equal(got, expected):
    tables, moves, count, status = expected
    for a, b in zip(got[0], tables):
        assert np.array_equal(a.cpu().numpy(), b)
    assert np.array_equal(got[1].cpu().numpy(), moves)
    assert int(got[2]) == count and int(got[3]) == status


def fork(parent, lengths, tables):
    p, n, *t = gpu([parent, lengths, *tables])
    equal((t, *cuda_ops.extension().paged_fork(p, n, *t)), sharing.paged_fork(parent, lengths, *tables))


def release(lengths, tables):
    n, *t = gpu([lengths, *tables])
    equal((t, *cuda_ops.extension().paged_release(n, *t)), sharing.paged_release(lengths, *tables))


def compact(tables):
    t = gpu(tables)
    equal((t, *cuda_ops.extension().paged_compact(*t)), sharing.paged_compact(*tables))


SIZES = [(1, 1, 100), (1, 3, 63), (1, 40, 5000), (7, 5, 64), (33, 9, 900), (600, 2, 70), (3, 0, 200), (1, 2, 0)]


@pytest.mark.parametrize("parents,children,longest", SIZES)
def test_fork_equals_the_definition(cuda, parents, children, longest):
    for seed in range(3):
        fork(*problem(seed, parents, children, longest, spare=seed, fork=True))


@pytest.mark.parametrize("parents,children,longest", SIZES)
def test_release_equals_the_definition(cuda, parents, children, longest):
    for seed in range(3):
        _, total, tables = problem(seed, parents, children, longest, spare=seed)
        rng = np.random.default_rng(seed + 100)
        cut = rng.integers(0, total + 1)
        for lengths in (cut, np.where(rng.random(len(cut)) < 0.3, 0, total), total * 0, total):
            release(lengths.astype(np.int32), tables)


@pytest.mark.parametrize("parents,children,longest", SIZES)
def test_compaction_equals_the_definition(cuda, parents, children, longest):
    for seed in range(3):
        compact(problem(seed, parents, children, longest, spare=seed * 700)[2])


def test_large_batches_and_pools(cuda):
    fork(*problem(4, 64, 255, 200, fork=True))
    _, total, tables = problem(5, 128, 127, 300, spare=70000)  # several passes over the freed blocks
    release((total // 3).astype(np.int32), tables)
    release((total * 0).astype(np.int32), tables)
    compact(tables)


def test_pools_of_a_few_blocks(cuda):
    for blocks in (1, 2, 3):
        none = (np.zeros(1, np.int32), np.full((1, 2), -1, np.int32), np.arange(blocks, dtype=np.int32),
                np.array([0, blocks, 0, 0], np.int32), np.zeros(blocks, np.int32))
        compact(none)
        one = (np.array([1], np.int32), np.array([[blocks - 1, -1]], np.int32), np.arange(blocks, dtype=np.int32),
               np.array([0, blocks - 1, 0, 0], np.int32), np.zeros(blocks, np.int32))
        compact(one)
        release(np.zeros(1, np.int32), one)


@pytest.mark.parametrize("fault", ["parent", "parent_low", "itself", "chain", "held", "longer", "negative", "short",
                                   "blocks", "head", "count", "stride"])
def test_refused_fork_changes_nothing(cuda, fault):
    parent, lengths, tables = problem(7, 4, 6, 700, fork=True)
    held, _, _, state, _ = tables
    child = int(np.flatnonzero(parent >= 0)[2])
    p = parent[child]
    lengths[p] = max(lengths[p], 65)
    held[p] = -(-lengths[p] // 64)
    lengths[child] = 65
    if fault == "parent":
        parent[child] = len(parent)
    elif fault == "parent_low":
        parent[child] = -2
    elif fault == "itself":
        parent[child] = child
    elif fault == "chain":
        parent[p] = int(np.flatnonzero(parent < 0)[0]) if np.flatnonzero(parent < 0)[0] != p else \
            int(np.flatnonzero(parent < 0)[1])
    elif fault == "held":
        held[child] = 1
    elif fault == "longer":
        lengths[child] = lengths[p] + 1
    elif fault == "negative":
        lengths[child] = -1
    elif fault == "short":
        held[p] -= 1
    elif fault == "blocks":
        state[1] = 0
    elif fault == "head":
        state[0] = -1
    elif fault == "count":
        state[1] = len(tables[2]) + 1
    elif fault == "stride":
        held[p] = tables[1].shape[1] + 1
    assert sharing.paged_fork(parent, lengths, *tables)[3] == 1
    fork(parent, lengths, tables)


@pytest.mark.parametrize("fault", ["length", "longer", "held", "blocks", "head", "count"])
def test_refused_release_changes_nothing(cuda, fault):
    _, total, tables = problem(8, 3, 8, 900)
    held, _, _, state, shares = tables
    b = int(np.argmax(np.where(shares[np.maximum(tables[1][:, 0], 0)] > 0, held, 0)))
    lengths = total.copy()
    lengths[b] = 33  # within a shared block
    if fault == "length":
        lengths[b] = -1
    elif fault == "longer":
        lengths[b] = held[b] * 64 + 1
    elif fault == "held":
        held[b] = -1
    elif fault == "blocks":
        state[1] = 0
    elif fault == "head":
        state[0] = len(tables[2])
    elif fault == "count":
        state[1] = -1
    assert sharing.paged_release(lengths, *tables)[3] == 1
    release(lengths, tables)


def test_blocks_that_were_lost_are_free_after_compaction(cuda):
    """Blocks that neither the ring nor an entry has, with counts left behind."""
    for spare in (9, 70000):
        tables = problem(15, 5, 4, 700, spare=spare)[2]
        held, table, _, state, shares = tables
        state[1] = 0
        mapped = np.unique(table[table >= 0])
        shares[np.setdiff1d(np.arange(len(shares)), mapped)[::2]] = 3
        compact(tables)


def test_refused_compaction_changes_nothing(cuda):
    tables = problem(9, 3, 3, 500)[2]
    tables[0][4] = tables[1].shape[1] + 1
    compact(tables)


def test_block_ids_outside_the_pool_are_reported(cuda):
    parent, lengths, tables = problem(10, 2, 5, 600, fork=True)
    lengths[:] = np.where(parent < 0, np.where(tables[0] > 0, 300, 0), 150)
    tables[0][:] = np.where((parent < 0) & (tables[0] > 0), 5, 0)
    tables[1][:, :5] = np.where(tables[0][:, None] > 0, np.arange(len(parent))[:, None] * 5 + np.arange(5), -1)
    p = parent[parent >= 0][0]
    tables[1][p, 1] = len(tables[2])      # a whole block
    fork(parent, lengths, tables)
    tables[1][p, 1], tables[1][p, 2] = p * 5 + 1, -4  # the copied one
    fork(parent, lengths, tables)
    tables[1][p, 2] = p * 5 + 2
    tables[2][tables[3][0]] = -9          # a free one
    fork(parent, lengths, tables)
    _, total, tables = problem(11, 2, 5, 600)
    b = int(np.argmax(tables[0]))
    tables[1][b, tables[0][b] - 1] = 1 << 30
    release((total * 0).astype(np.int32), tables)
    compact(tables)
    _, total, tables = problem(12, 1, 4, 600)
    tables[4][:] = 0                      # counts that miss the shares
    release((total * 0).astype(np.int32), tables)


@pytest.mark.parametrize("layers", [0, 1, 3, 33])
def test_copies_are_bit_for_bit(cuda, layers):
    rng = np.random.default_rng(layers)
    rows = 64 * 40
    pools = [torch.randn((rows, w), device="cuda").to(t) for _ in range(layers)
             for w, t in ((576, torch.bfloat16), (128, torch.bfloat16), (4, torch.float32))]
    gens = [torch.randint(0, 9, (rows,), device="cuda") for _ in range(max(layers, 1))]
    block = rng.permutation(40)
    moves = np.array([(block[i] * 64, block[20 + i] * 64, n, 0) for i, n in enumerate((64, 1, 63, 0, 17, 33, 64, 64))]
                     + [(block[0] * 64, block[30] * 64, 64, 0)], np.int32)  # one source twice
    for count in (0, 1, 5, len(moves)):
        expected = sharing.paged_copy([p.view(torch.int16).cpu().numpy() for p in pools], [g.cpu().numpy() for g in gens],
                                      moves, count)
        status = cuda_ops.extension().paged_copy(pools, gens, *gpu([moves, np.array([count], np.int32)]))
        assert int(status) == 0
        for a, b in zip(pools, expected[0]):
            assert np.array_equal(a.view(torch.int16).cpu().numpy(), b)
        for a, b in zip(gens, expected[1]):
            assert np.array_equal(a.cpu().numpy(), b)


def test_bad_moves_are_reported_and_skipped(cuda):
    pool = torch.arange(64 * 4 * 8, device="cuda", dtype=torch.int16).view(256, 8)
    gens = torch.zeros(256, dtype=torch.int64, device="cuda")
    good = (0, 64, 3, 0)
    for bad in ((-1, 128, 2, 0), (0, -64, 1, 0), (200, 128, 64, 0), (0, 255, 2, 0), (0, 128, 65, 0), (0, 128, -1, 0)):
        before = pool.clone()
        status = cuda_ops.extension().paged_copy([pool], [gens], *gpu([np.array([bad, good], np.int32),
                                                                       np.array([2], np.int32)]))
        assert int(status) == 1
        before[64:67] = before[0:3]
        assert torch.equal(pool, before)
    before = gens.clone()
    for count in (-1, 3):
        status = cuda_ops.extension().paged_copy([pool], [gens], *gpu([np.array([good, good], np.int32),
                                                                       np.array([count], np.int32)]))
        assert int(status) == 1 and torch.equal(gens, before)


def test_a_graph_of_the_calls_and_another_stream(cuda):
    """Captured once, replayed on other lengths; the run on a side stream gives the same."""
    ext = cuda_ops.extension()
    parent, lengths, tables = problem(13, 3, 7, 900, spare=60, fork=True)
    ended = np.where(parent >= 0, 0, lengths).astype(np.int32)
    rows = len(tables[2]) * 64
    for graphed in (True, False):
        p, n, e, *t = gpu([parent, lengths, ended, *tables])
        pool = torch.arange(rows * 8, device="cuda", dtype=torch.int32).view(rows, 8)
        gens = torch.zeros(rows, dtype=torch.int64, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")

        def step():
            moves, count, _ = ext.paged_fork(p, n, *t, status=status)
            ext.paged_copy([pool], [gens], moves, count, status=status)
            cut, cuts, _ = ext.paged_release(e, *t, status=status)
            ext.paged_copy([pool], [gens], cut, cuts, status=status)
            more, counts, _ = ext.paged_compact(*t, status=status)
            ext.paged_copy([pool], [gens], more, counts, status=status)
            return moves, count, more, counts

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        if graphed:
            keep = [x.clone() for x in (*t, pool, gens)]
            step()  # loads the kernels before the capture
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = step()
            for x, y in zip((*t, pool, gens), keep):
                x.copy_(y)
        expected, ref_pool, ref_gens = tables, pool.cpu().numpy(), gens.cpu().numpy()
        now = lengths
        for i in range(4):
            if graphed:
                graph.replay()
            else:
                with torch.cuda.stream(stream):
                    outs = step()
                torch.cuda.current_stream().wait_stream(stream)
            expected, moves, count, s0 = sharing.paged_fork(parent, now, *expected)
            (ref_pool,), (ref_gens,) = sharing.paged_copy([ref_pool], [ref_gens], moves, count)
            expected, cut, cuts, s1 = sharing.paged_release(ended, *expected)
            (ref_pool,), (ref_gens,) = sharing.paged_copy([ref_pool], [ref_gens], cut, cuts)
            expected, more, counts, s2 = sharing.paged_compact(*expected)
            (ref_pool,), (ref_gens,) = sharing.paged_copy([ref_pool], [ref_gens], more, counts)
            assert s0 == s1 == s2 == 0 == int(status)
            for a, b in zip((*t, *outs, pool, gens), (*expected, moves, count, more, counts, ref_pool, ref_gens)):
                assert np.array_equal(a.cpu().numpy().squeeze(), np.squeeze(b))
            now = np.where(parent >= 0, np.minimum(now, now // 2 + i), now).astype(np.int32)
            n.copy_(torch.from_numpy(now))


def test_checked_calls_and_refusals(cuda):
    parent, lengths, tables = problem(14, 2, 3, 300, fork=True)
    p, n, *t = gpu([parent, lengths, *tables])
    moves, count = cuda_ops.paged_fork(p, n, *t)
    pool, gens = torch.zeros((len(tables[2]) * 64, 576), device="cuda").bfloat16(), torch.zeros(
        len(tables[2]) * 64, dtype=torch.int64, device="cuda")
    cuda_ops.paged_copy([pool], [gens], moves, count)
    assert int(gens.sum()) == int(moves[:, 2].sum())
    cuda_ops.paged_release(n, *t)
    cuda_ops.paged_compact(*t)
    with pytest.raises(cuda_ops.ValidationError):  # the children hold blocks now
        cuda_ops.paged_fork(p, n, *t)
    with pytest.raises(cuda_ops.ValidationError):
        cuda_ops.paged_release(n - 1000, *t)
    ext = cuda_ops.extension()
    for bad in ((p.long(), n, *t), (p[:2], n, *t), (p, n[:2], *t), (p, n, t[0], t[1][:2], *t[2:]),
                (p, n, *t[:4], t[4][:3]), (p, n, t[0], t[1].cpu(), *t[2:]), (p, n, *t[:3], t[3][:3], t[4])):
        with pytest.raises(RuntimeError):
            ext.paged_fork(*bad)
    with pytest.raises(RuntimeError):
        ext.paged_release(n.float(), *t)
    with pytest.raises(RuntimeError):
        ext.paged_compact(*t[:4], t[4].long())
    for bad in (([pool[:64], pool], [gens], moves, count), ([pool], [gens[:5]], moves, count),
                ([pool], [gens.int()], moves, count), ([pool[:, :100]], [gens], moves, count),
                ([pool], [gens], moves[:, :3].contiguous(), count), ([pool], [gens], moves, moves),
                ([torch.zeros((len(pool), 3), device="cuda")], [gens], moves, count),
                ([pool.float().requires_grad_()], [gens], moves, count)):
        with pytest.raises(RuntimeError):
            ext.paged_copy(*bad)


def test_copies_in_several_launches_are_refused_as_a_whole(cuda):
    """More pools and generations than a launch takes: a bad one at the end, or one given twice."""
    pools = [torch.arange(128 * 8, device="cuda", dtype=torch.int16).view(128, 8) for _ in range(70)]
    gens = [torch.zeros(128, dtype=torch.int64, device="cuda") for _ in range(70)]
    moves = gpu([np.array([(0, 64, 5, 0)], np.int32), np.array([1], np.int32)])
    before = pools[0].clone()
    narrow = torch.zeros((128, 4), device="cuda", dtype=torch.int16)
    misplaced = torch.zeros(128 * 8 + 1, device="cuda", dtype=torch.int16)[1:].view(128, 8)
    for bad in ((pools + [narrow], gens), (pools + [misplaced], gens), (pools, gens + gens[:1]), (pools, gens[:1] * 2)):
        with pytest.raises(RuntimeError):
            cuda_ops.extension().paged_copy(*bad, *moves)
        assert torch.equal(pools[0], before) and not gens[0].any()
    assert int(cuda_ops.extension().paged_copy(pools, gens, *moves)) == 0
    before[64:69] = before[:5]
    for p, g in zip(pools, gens):
        assert torch.equal(p, before) and int(g.sum()) == int(g[64:69].sum()) == 5
