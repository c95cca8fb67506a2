"""64-bit definitions of the operators around the paged decode path (test infrastructure only).

Block tables and slot maps, rotary positions, attention of drafted tokens and
sampling, each written from its formula; none has a counterpart in the
reference's own sources.
"""
from __future__ import annotations

import numpy as np

BLOCK, V_DIM = 64, 512


def paged_plan(lengths, new_tokens, held, table, ring, state, tokens, shares=None):
    """New (held, table, ring, state), the token map and the status of one plan.

    With shares: a plan that maps a new token to a block with shares, or gives one back, is refused."""
    held, table, ring, state = (np.array(a) for a in (held, table, ring, state))
    batch, blocks = len(lengths), len(ring)
    head, count = int(state[0]), int(state[1])
    total = lengths.astype(np.int64) + new_tokens
    need = -(-total // BLOCK)
    takes = int(np.maximum(need - held, 0).sum())
    gives = int(np.maximum(held - need, 0).sum())
    maps = [np.full(tokens, -1, np.int32) for _ in range(3)]
    if ((lengths < 0) | (new_tokens < 0) | (total > table.shape[1] * BLOCK) | (held < 0) |
            (held > table.shape[1])).any() or int(new_tokens.sum()) > tokens or takes > count or \
            not 0 <= head < blocks or count < 0 or count + gives > blocks or \
            shares is not None and meets_shared(lengths, new_tokens, need, held, table, shares):
        return held, table, ring, state, maps, np.zeros(batch + 1, np.int32), lengths.copy(), 1
    status, i = 0, 0
    tail = head + count
    for b in range(batch):
        for j in range(held[b], need[b]):
            block = ring[head % blocks]
            head += 1
            if not 0 <= block < blocks:
                block, status = -1, 1
            table[b, j] = block
        for j in range(need[b], held[b]):
            block = table[b, j]
            if not 0 <= block < blocks:
                block, status = -1, 1
            ring[tail % blocks] = block
            tail += 1
            table[b, j] = -1
        for p in range(lengths[b], total[b]):
            block = table[b, p // BLOCK]
            if 0 <= block < blocks:
                slot = block * BLOCK + p % BLOCK
            else:
                slot, status = -1, 1
            maps[0][i], maps[1][i], maps[2][i] = b, p, slot
            i += 1
    state[0], state[1] = head % blocks, count - takes + gives
    cu = np.concatenate([[0], np.cumsum(new_tokens)]).astype(np.int32)
    return need.astype(np.int32), table, ring, state, maps, cu, total.astype(np.int32), status


def meets_shared(lengths, new_tokens, need, held, table, shares):
    """Whether a held block that new tokens go to, or that is given back, has shares."""
    for b, n in enumerate(lengths):
        touched = {p // BLOCK for p in range(n, n + new_tokens[b])} | set(range(need[b], held[b]))
        blocks = [table[b, j] for j in touched if j < held[b]]
        if any(shares[i] > 0 for i in blocks if 0 <= i < len(shares)):
            return True
    return False


def rope(x, positions, frequencies, offset, interleaved, mscale=1.0, inverse=False):
    """x [tokens, heads, width] float64 -> rotated copy (rows of position -1 unchanged)."""
    y = np.array(x, np.float64)
    pairs = len(frequencies)
    angle = positions.astype(np.float64)[:, None] * np.asarray(frequencies, np.float64)
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None] * (-1 if inverse else 1)
    i = np.arange(pairs)
    a, b = (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + i + pairs)
    xa, xb = y[..., a], y[..., b]
    ya, yb = mscale * (xa * cos - xb * sin), mscale * (xb * cos + xa * sin)
    real = (positions >= 0)[:, None, None]
    y[..., a], y[..., b] = np.where(real, ya, xa), np.where(real, yb, xb)
    return y


def sample(logits, temperature, top_k, top_p, min_p, uniform):
    """(token, chance) of one row of float64 logits; -1, 0 when nothing can be drawn."""
    top = logits.max()
    if top == -np.inf:
        return -1, 0.0
    if temperature == 0:
        return int(np.argmax(logits)), 1.0
    weight = np.exp((logits - top) / np.float64(temperature))
    order = np.lexsort((np.arange(len(logits)), -logits))
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(weight[order])
        order = order[:max(1, int((mass - weight[order] < np.float64(top_p) * mass[-1]).sum()))]
    order = order[weight[order] >= np.float64(min_p)]
    kept = np.sort(order)
    sums = np.cumsum(weight[kept])
    at = int(np.searchsorted(sums, np.float64(uniform) * sums[-1], side="right"))
    token = int(kept[min(at, len(kept) - 1)])
    return token, weight[token] / sums[-1]


def tree_attention(q, keys, context, masks, sink, scale):
    """Drafted nodes of one sequence: q [nodes, heads, 576], keys [context + nodes, 576]
    float64, masks int (bit j: the node sees node j) -> out [nodes, heads, 512], and the
    logarithm of each row's sum (-inf when it sees nothing and has no sink)."""
    nodes, heads, _ = q.shape
    out = np.zeros((nodes, heads, V_DIM))
    lse = np.full((nodes, heads), -np.inf)
    for n in range(nodes):
        seen = list(range(context)) + [context + j for j in range(nodes) if int(masks[n]) >> j & 1]
        s = scale * (q[n] @ keys[seen].T)
        if sink is not None:
            s = np.concatenate([s, np.asarray(sink, np.float64)[:, None]], 1)
        if s.shape[1] == 0:
            continue
        top = s.max(1, keepdims=True)
        e = np.exp(s - top)
        total = e.sum(1, keepdims=True)
        out[n] = (e[:, :len(seen)] / total) @ keys[seen][:, :V_DIM]
        lse[n] = (top + np.log(total))[:, 0]
    return out, lse
