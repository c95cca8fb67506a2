"""Blocks that several requests map, and the attention over common prompts, without a GPU:
refusals of the C ABI, the definitions that the GPU tests rest on, and rules of the source."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest

from oracle import serving, sharing
from deepseekrpc_b200 import _native

P = 256  # a pointer that passes the alignment checks; nothing is launched


def fork(n, parent=P, lengths=P, held=P, table=P, stride=4, ring=P, state=P, shares=P, blocks=8, moves=P, count=P,
         err=P, batch=2):
    return n.dsr_paged_fork(parent, lengths, held, table, stride, ring, state, shares, blocks, moves, count, err, batch,
                            None)


def release(n, lengths=P, held=P, table=P, stride=4, shares=P, blocks=8, moves=P, ws=P, ws_bytes=1 << 40, err=P,
            batch=2):
    return n.dsr_paged_release(lengths, held, table, stride, P, P, shares, blocks, moves, P, ws, ws_bytes, err, batch,
                               None)


def compact(n, held=P, table=P, stride=4, shares=P, blocks=8, moves=P, ws=P, ws_bytes=1 << 40, err=P, batch=2):
    return n.dsr_paged_compact(held, table, stride, P, P, shares, blocks, moves, P, ws, ws_bytes, err, batch, None)


def copy(n, pools=(P, 512), row_bytes=(1152, 256), gens=(P,), rows=64, moves=P, count=P, room=4, err=P):
    data = (ctypes.c_void_p * max(len(pools), 1))(*pools)
    widths = (ctypes.c_int64 * max(len(row_bytes), 1))(*row_bytes)
    bumps = (ctypes.c_void_p * max(len(gens), 1))(*gens)
    return n.dsr_paged_copy(data, widths, len(pools), bumps, len(gens), rows, moves, count, room, err, None)


def prefix(n, q=P, dtype=0, pool=P, blocks=8, table=P, rows=3, stride=4, context=P, cu=P, mask=P, most=4, prefix=P,
           holder=P, scale=1.0, out=P, out_dtype=0, ws=P, ws_bytes=1 << 40, err=P, batch=2, nodes=4, heads=16):
    return n.dsr_prefix_mla_decode(q, dtype, pool, blocks, table, rows, stride, context, cu, mask, most, prefix, holder, None,
                                   scale, out, out_dtype, None, ws, ws_bytes, err, batch, nodes, heads, None)


@pytest.mark.parametrize("call", [
    *(lambda n, k=k: prefix(n, **{k: None}) for k in ("q", "pool", "table", "context", "cu", "mask", "prefix", "holder",
                                                      "out", "ws", "err")),
    lambda n: prefix(n, dtype=2), lambda n: prefix(n, out_dtype=5), lambda n: prefix(n, blocks=0),
    lambda n: prefix(n, rows=1), lambda n: prefix(n, rows=1 << 31), lambda n: prefix(n, stride=0),
    lambda n: prefix(n, most=0), lambda n: prefix(n, most=65), lambda n: prefix(n, scale=0.0),
    lambda n: prefix(n, scale=float("nan")), lambda n: prefix(n, out=264), lambda n: prefix(n, q=264),
    lambda n: prefix(n, ws=128), lambda n: prefix(n, ws_bytes=1000), lambda n: prefix(n, batch=0),
    lambda n: prefix(n, batch=16385, rows=20000), lambda n: prefix(n, nodes=0), lambda n: prefix(n, nodes=(1 << 20) + 1),
    lambda n: prefix(n, heads=24), lambda n: prefix(n, heads=0),
    *(lambda n, k=k: fork(n, **{k: None}) for k in ("parent", "lengths", "held", "table", "ring", "state", "shares",
                                                    "moves", "count", "err")),
    lambda n: fork(n, stride=0), lambda n: fork(n, stride=1 << 25), lambda n: fork(n, blocks=0),
    lambda n: fork(n, batch=0), lambda n: fork(n, batch=16385), lambda n: fork(n, moves=264),
    *(lambda n, k=k: release(n, **{k: None}) for k in ("lengths", "held", "table", "shares", "moves", "ws", "err")),
    lambda n: release(n, ws=128), lambda n: release(n, ws_bytes=100), lambda n: release(n, batch=16385),
    lambda n: release(n, blocks=1 << 25),
    *(lambda n, k=k: compact(n, **{k: None}) for k in ("held", "table", "shares", "moves", "ws", "err")),
    lambda n: compact(n, ws_bytes=100), lambda n: compact(n, ws=264), lambda n: compact(n, batch=0),
    lambda n: compact(n, blocks=8388609),
    lambda n: copy(n, moves=None), lambda n: copy(n, moves=8), lambda n: copy(n, count=None), lambda n: copy(n, err=None),
    lambda n: copy(n, pools=(P, None)), lambda n: copy(n, pools=(P, 520)), lambda n: copy(n, row_bytes=(1152, 8)),
    lambda n: copy(n, row_bytes=(0, 256)), lambda n: copy(n, row_bytes=(1152, 65552)), lambda n: copy(n, gens=(None,)),
    lambda n: copy(n, rows=0), lambda n: copy(n, rows=1 << 31), lambda n: copy(n, room=-1),
    lambda n: copy(n, pools=(P,) * 65, row_bytes=(16,) * 65), lambda n: copy(n, gens=(P,) * 65),
    lambda n: copy(n, gens=(P, 512, P)),
])
def test_host_side_validation_refuses_without_touching_a_device(call):
    lib = _native.library()
    assert call(lib) == _native.DSR_EINVAL
    assert _native.last_error()


def test_copy_of_no_moves_or_no_pools_launches_nothing():
    lib = _native.library()
    assert copy(lib, room=0) == _native.DSR_OK
    assert copy(lib, pools=(), row_bytes=(), gens=()) == _native.DSR_OK


def test_workspaces_are_pure_host_functions():
    lib = _native.library()
    assert lib.dsr_paged_release_workspace_bytes(0, 8) == lib.dsr_paged_compact_workspace_bytes(0) == 0
    assert lib.dsr_paged_release_workspace_bytes(16384, 1000) >= 16385 * 4 + 1000 // 8
    assert lib.dsr_paged_compact_workspace_bytes(1000) >= 1000 // 8
    assert lib.dsr_prefix_mla_workspace_bytes(0, 1, 16) == lib.dsr_prefix_mla_workspace_bytes(1, 0, 16) == 0
    # partials of all rows, of the prompts' and the requests' own parts
    assert lib.dsr_prefix_mla_workspace_bytes(64, 64, 128) >= 2 * 64 * 128 * 514 * 4


def test_rules_of_the_pairs_waits():
    """What no run can show.  A warp has one answer to a wait: outside the helper that asks all
    lanes nothing waits for a pair's barrier.  Softmax warps meet in named barriers, which know
    no limit: one whose wait gives up says so in the next vote and does not leave by itself."""
    source = Path(__file__).resolve().parent.parent / "deepseekrpc_b200" / "csrc" / "prefix_mla.cu"
    text = re.sub(r"//[^\n]*", "", source.read_text())
    helper = re.search(r"bool pair_wait_warp\([^{]*\{(.*?)\n\}", text, re.S)
    assert helper and "__all_sync(~0u, pair_wait(" in helper.group(1)
    assert len(re.findall(r"\bpair_wait\(", text)) == 2  # its definition, and there
    softmax = text[text.index("if (warp < 8) {"):text.index("} else if (warp == 8) {")]
    leaves = [m.start() for m in re.finditer(r"if \(!ok\) break;", softmax)]
    assert len(leaves) == 3
    for at in leaves:  # behind a vote of the rows' warps
        assert "rows_sync(pack," in softmax[:at].rstrip().rsplit("\n", 1)[-1], softmax[at - 120:at]
    assert "multicast" not in re.sub(r"tcgen05\.commit[^;]*;", "", text)  # no copy to several CTAs


def consistent(held, table, ring, state, shares):
    """Every block is free once, or mapped 1 + shares times."""
    blocks = len(ring)
    mapped = np.zeros(blocks, np.int64)
    for b, n in enumerate(held):
        assert (table[b, :n] >= 0).all() and (table[b, n:] == -1).all()
        np.add.at(mapped, table[b, :n], 1)
    free = [int(ring[(state[0] + i) % blocks]) for i in range(state[1])]
    assert sorted(free + np.flatnonzero(mapped).tolist()) == list(range(blocks))
    assert np.array_equal(shares, np.maximum(mapped - 1, 0))


def test_definitions_keep_every_block_and_every_request_its_rows():
    """Requests grow, fork, are cut and moved together; each has the tokens it should."""
    rng = np.random.default_rng(1)
    batch, blocks, stride = 9, 120, 10
    lengths, held = np.zeros(batch, np.int32), np.zeros(batch, np.int32)
    tables = (held, np.full((batch, stride), -1, np.int32), rng.permutation(blocks).astype(np.int32),
              np.array([0, blocks, 0, 0], np.int32), np.zeros(blocks, np.int32))
    pool, gens = np.full((blocks * 64, 1), -1, np.int64), np.zeros(blocks * 64, np.int64)
    tokens, stamp = [[] for _ in range(batch)], 0
    for _ in range(60):
        # cut (some end), with the exchange of shared last blocks
        kept = [int(rng.integers(0, n + 1)) if rng.random() < 0.4 else n for n in lengths]
        lengths = np.array([0 if rng.random() < 0.15 else k for k in kept], np.int32)
        *done, status = sharing.paged_release(lengths, *tables)
        tables, moves, count = done
        assert status == 0
        (pool,), (gens,) = sharing.paged_copy([pool], [gens], moves, count)
        tokens = [t[:n] for t, n in zip(tokens, lengths)]
        consistent(*tables)
        # fork into the empty ones
        parent = np.full(batch, -1, np.int32)
        full = [b for b in range(batch) if lengths[b] > 0]
        for b in range(batch):
            if lengths[b] == 0 and full and rng.random() < 0.7:
                parent[b] = rng.choice(full)
                lengths[b] = rng.integers(0, lengths[parent[b]] + 1)
                tokens[b] = tokens[parent[b]][:lengths[b]]
        *done, status = sharing.paged_fork(parent, lengths, *tables)
        tables, moves, count = done
        assert status == 0
        (pool,), (gens,) = sharing.paged_copy([pool], [gens], moves, count)
        consistent(*tables)
        if rng.random() < 0.3:
            *done, status = sharing.paged_compact(*tables)
            tables, moves, count = done
            assert status == 0
            (pool,), (gens,) = sharing.paged_copy([pool], [gens], moves, count)
            consistent(*tables)
            used = blocks - int(tables[3][1])
            assert all(tables[1][b, j] < used for b in range(batch) for j in range(tables[0][b]))
        # grow
        new = rng.integers(0, 70, batch).astype(np.int32)
        new[lengths + new > 6 * 64] = 0
        *first, shares = tables
        *first, maps, cu, visible, status = serving.paged_plan(lengths, new, *first, int(new.sum()))
        tables = (*first, shares)
        assert status == 0
        for s, _, slot in zip(*maps):
            pool[slot] = stamp
            tokens[s].append(stamp)
            stamp += 1
        lengths = (lengths + new).astype(np.int32)
        consistent(*tables)
        for b in range(batch):
            at = [tables[1][b, p // 64] * 64 + p % 64 for p in range(lengths[b])]
            assert pool[at, 0].tolist() == tokens[b]
