"""Definitions of the operators on blocks that several requests map (test infrastructure only).

Forking, cutting and compacting the requests of a paged cache, block by block in plain
loops, and the copies of rows that they name; none has a counterpart in the reference's
own sources.
"""
from __future__ import annotations

import numpy as np

BLOCK = 64
NO_MOVE = (-1, -1, 0, 0)


def _state_fits(held, table, ring, state):
    blocks = len(ring)
    return 0 <= state[0] < blocks and 0 <= state[1] <= blocks and not ((held < 0) | (held > table.shape[1])).any()


def _moves(entries, room):
    out = np.array([NO_MOVE] * room, np.int32).reshape(room, 4)
    for i, entry in enumerate(entries):
        out[i] = entry
    return out


def paged_fork(parent, lengths, held, table, ring, state, shares):
    """New (held, table, ring, state, shares), moves, count and status."""
    held, table, ring, state, shares = (np.array(a) for a in (held, table, ring, state, shares))
    batch, blocks = len(parent), len(ring)
    tables = held, table, ring, state, shares
    children = [b for b in range(batch) if parent[b] != -1]
    fits = 0 <= state[0] < blocks and 0 <= state[1] <= blocks
    for b in children:
        p = parent[b]
        fits = fits and 0 <= p < batch and p != b and parent[p] == -1 and held[b] == 0
        fits = fits and 0 <= held[p] <= table.shape[1] and 0 <= lengths[b] <= lengths[p] <= int(held[p]) * BLOCK
    takes = sum(int(lengths[b]) % BLOCK != 0 for b in children)
    if not fits or takes > state[1]:
        return tables, _moves([], batch), 0, 1
    status, moves, head = 0, [], int(state[0])
    good = lambda block: 0 <= block < blocks  # noqa: E731
    for b in children:
        n, p = int(lengths[b]), parent[b]
        for j in range(-(-n // BLOCK)):
            block = table[p, j]
            if not good(block):
                status = 1
            if j < n // BLOCK:
                table[b, j] = block if good(block) else -1
                if good(block):
                    shares[block] += 1
            else:
                fresh = ring[head % blocks]
                head += 1
                if not good(fresh):
                    status = 1
                table[b, j] = fresh if good(fresh) else -1
                moves.append((block * BLOCK, fresh * BLOCK, n % BLOCK, 0) if good(block) and good(fresh) else NO_MOVE)
        held[b] = -(-n // BLOCK)
    state[0], state[1] = head % blocks, state[1] - takes
    return tables, _moves(moves, batch), takes, status


def paged_release(lengths, held, table, ring, state, shares):
    """New (held, table, ring, state, shares), moves, count and status."""
    held, table, ring, state, shares = (np.array(a) for a in (held, table, ring, state, shares))
    batch, blocks = len(lengths), len(ring)
    tables = held, table, ring, state, shares
    need = -(-lengths.astype(np.int64) // BLOCK)
    good = lambda block: 0 <= block < blocks  # noqa: E731
    fits = _state_fits(held, table, ring, state) and not ((lengths < 0) | (need > held)).any()
    cut = [b for b in range(batch) if fits and lengths[b] % BLOCK and good(table[b, need[b] - 1])
           and shares[table[b, need[b] - 1]] > 0]
    if not fits or len(cut) > state[1]:
        return tables, _moves([], batch), 0, 1
    status, moves, dropped = 0, [], []
    head, count = int(state[0]), int(state[1])
    for b in range(batch):
        if lengths[b] % BLOCK and not good(table[b, need[b] - 1]):
            status = 1
        if b in cut:
            source, fresh = table[b, need[b] - 1], ring[head % blocks]
            head += 1
            if not good(fresh):
                status = 1
            moves.append((source * BLOCK, fresh * BLOCK, lengths[b] % BLOCK, 0) if good(fresh) else NO_MOVE)
            table[b, need[b] - 1] = fresh if good(fresh) else -1
            dropped.append(source)
        for j in range(need[b], held[b]):
            dropped.append(table[b, j])
            table[b, j] = -1
        held[b] = need[b]
    for block in dropped:
        if good(block):
            status = status or int(shares[block] < 0)
            shares[block] -= 1
        else:
            status = 1
    free = np.flatnonzero(shares < 0)
    for i, block in enumerate(free):
        ring[(int(state[0]) + count + i) % blocks] = block
        shares[block] = 0
    state[0], state[1] = head % blocks, min(count - len(cut) + len(free), blocks)
    return tables, _moves(moves, batch), len(cut), status


def paged_compact(held, table, ring, state, shares):
    """New (held, table, ring, state, shares), moves, count and status."""
    held, table, ring, state, shares = (np.array(a) for a in (held, table, ring, state, shares))
    blocks, room = len(ring), max(len(ring) // 2, 1)
    tables = held, table, ring, state, shares
    if ((held < 0) | (held > table.shape[1])).any():
        return tables, _moves([], room), 0, 1
    mapped = [(b, j) for b in range(len(held)) for j in range(held[b])]
    status = int(any(not 0 <= table[at] < blocks for at in mapped))
    live = sorted({int(table[at]) for at in mapped if 0 <= table[at] < blocks})
    used = len(live)
    holes = sorted(set(range(used)) - set(live))
    target = dict(zip([i for i in live if i >= used], holes))
    for at in mapped:
        table[at] = target.get(int(table[at]), table[at])
    for source, to in target.items():
        shares[to], shares[source] = shares[source], 0
    shares[used:] = 0
    ring[:] = -1
    ring[:blocks - used] = np.arange(used, blocks)
    state[0], state[1] = 0, blocks - used
    return tables, _moves([(s * BLOCK, t * BLOCK, BLOCK, 0) for s, t in target.items()], room), len(target), status


def paged_copy(pools, generations, moves, count):
    """Changed copies of the pools and generations."""
    pools, generations = [np.array(p) for p in pools], [np.array(g) for g in generations]
    for source, to, rows, _ in moves[:count]:
        for p in pools:
            p[to:to + rows] = p[source:source + rows]
        for g in generations:
            g[to:to + rows] += 1
    return pools, generations
