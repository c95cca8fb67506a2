"""What the operators of a paged cache with shared blocks cost.

Requests that continue one prompt share its blocks: `paged_fork` gives a child its
parent's whole blocks and a copy of the last, `paged_release` shortens or ends
requests whose blocks others may map, `paged_compact` moves the blocks in use to the
lowest ids, `paged_copy` moves the rows that these three name, and `prefix_mla_decode`
attends from all requests of a prompt over its rows at once.  `run` computes a case
either with elementary torch operations (own = False) or with this package's kernels.
"""
from __future__ import annotations

import math

import torch

own = False  # True: `run` calls this package's operators

BLOCK, KV, DV, INDEX = 64, 576, 512, 128
SCALE = 1 / math.sqrt(192)


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one request branches once in the middle of a block: latency alone
        dict(name="fork 1", op="fork", parents=1, children=1, low=4001, high=4001, layers=1),
        # 64 requests continue one cached prompt
        dict(name="fork 64 of one prompt", op="fork", parents=1, children=64, low=32801, high=32801, layers=1),
        # many answers to ragged prompts, caches of four layers
        dict(name="fork 33x15", op="fork", parents=33, children=15, low=500, high=16000, layers=4),
        # eight beams rolled back into what they share
        dict(name="trim 8", op="trim", parents=1, children=8, low=4100, high=4100, layers=1),
        # a large batch of which every request is cut somewhere, or ends
        dict(name="trim 64x7", op="trim", parents=64, children=7, low=1000, high=32000, layers=1),
        # a small pool of a few requests
        dict(name="compact 300", op="compact", parents=5, children=3, low=300, high=2000, blocks=300, layers=1),
        # a large pool half in use, its blocks anywhere
        dict(name="compact 16384", op="compact", parents=64, children=3, low=1000, high=14000, blocks=16384, layers=1),
        # two answers to a short prompt: latency
        dict(name="prefix 2 of 4K", op="prefix", batch=2, runs=1, nodes_low=1, nodes_high=1, heads=16,
             prefix_low=4096, prefix_high=4096, own_low=1, own_high=64, sink=False),
        # drafted tokens of ragged requests that continue one of five prompts
        dict(name="prefix 23 of 5 prompts", op="prefix", batch=23, runs=5, nodes_low=1, nodes_high=6, heads=32,
             prefix_low=1001, prefix_high=24000, own_low=1, own_high=700, sink=True),
        # a batch of answers to one long prompt
        dict(name="prefix 64 of 32K", op="prefix", batch=64, runs=1, nodes_low=1, nodes_high=1, heads=128,
             prefix_low=32768, prefix_high=32768, own_low=1, own_high=1500, sink=True),
        # a large batch, a prompt of documents
        dict(name="prefix 256 of 64K", op="prefix", batch=256, runs=1, nodes_low=1, nodes_high=1, heads=64,
             prefix_low=65499, prefix_high=65499, own_low=1, own_high=1000, sink=False),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("fork", "trim", "compact", "prefix", "prefix"))
    if op == "prefix":
        while True:
            batch, nodes, heads = _log(rng, 1, 256), rng.choice((1, 1, rng.randint(2, 12))), rng.choice((16, 32, 64, 128))
            high, most = _log(rng, 64, 65536), _log(rng, 1, 4000)
            runs = min(batch, _log(rng, 1, 12))
            low = rng.choice((high, high // 8))
            # products and cached rows at most those of the largest listed case
            if (batch * nodes * heads * (high + most) <= 256 * 64 * 66000 and batch * nodes * heads <= 32768
                    and batch * most + runs * high <= 400000):
                return dict(op=op, batch=batch, runs=runs, nodes_low=rng.choice((1, nodes)), nodes_high=nodes, heads=heads,
                            prefix_low=low, prefix_high=high, own_low=1, own_high=most, sink=rng.random() < 0.5)
    while True:
        parents, children, high = _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 1, 40000)
        low, layers = rng.choice((high, max(1, high // 16))), rng.choice((1, 1, 2, 4))
        blocks = parents * (high // BLOCK + 3) + 3 * parents * children
        if op == "compact":
            blocks = round(blocks * rng.uniform(1.1, 3))
        if parents * children <= 512 and blocks * layers <= 16384:
            case = dict(op=op, parents=parents, children=children, low=low, high=high, layers=layers)
            return dict(case, blocks=blocks) if op == "compact" else case


# ----------------------------------------------------------------- the inputs
def _between(low, high, n, gen):
    return torch.randint(low, high + 1, (n,), generator=gen, dtype=torch.int64)


def _spread(low, high, n):
    """Ragged counts that are the same for every seed: the outputs' shapes go by them."""
    return low + (torch.arange(n) * 1237 + high - low) % (high - low + 1)


def _i32(t):
    return t.to(torch.int32).cuda()


def _flat(parts):
    """The tensors as views of one buffer, each from a 16-byte boundary."""
    padded = [torch.nn.functional.pad(p.reshape(-1), (0, -p.numel() % 4)) for p in parts]
    store = _i32(torch.cat(padded))
    views, at = [], 0
    for p, whole in zip(parts, padded):
        views.append(store[at:at + p.numel()].view(p.shape))
        at += whole.numel()
    return store, views


def _pages(case, s, cpu, gpu):
    """Parents in the first rows, their children behind them; a pool for every layer."""
    parents, each = case["parents"], case["children"]
    n, requests = parents * each, parents * (each + 1)
    lengths = _between(case["low"], case["high"], parents, cpu)
    source = torch.arange(n) // each
    length_c = lengths[source] if case["low"] == case["high"] else 1 + (
        torch.rand(n, generator=cpu) * lengths[source]).long().clamp(max=lengths[source] - 1)
    held_p, whole = (lengths + BLOCK - 1) // BLOCK, length_c // BLOCK
    # a child beyond the fork: its own tail, and a block or so more
    grown = length_c + _between(0, BLOCK, n, cpu) if case["op"] != "fork" else length_c
    held_c = (grown + BLOCK - 1) // BLOCK
    stride = case["high"] // BLOCK + 3
    blocks = case.get("blocks") or parents * (case["high"] // BLOCK + 3) + 3 * n
    ids = torch.randperm(blocks, generator=cpu)
    j = torch.arange(stride)[None]
    at = torch.cumsum(held_p, 0) - held_p
    table_p = torch.where(j < held_p[:, None], ids[torch.where(j < held_p[:, None], at[:, None] + j, 0)], -1)
    used = int(held_p.sum())
    if case["op"] == "fork":
        table_c, held = torch.full((n, stride), -1), torch.cat([held_p, torch.zeros(n, dtype=torch.int64)])
    else:
        private = held_c - whole
        first = used + torch.cumsum(private, 0) - private
        own_ids = ids[torch.where((j >= whole[:, None]) & (j < held_c[:, None]),
                                  first[:, None] + j - whole[:, None], 0)]
        table_c = torch.where(j < whole[:, None], table_p[source], torch.where(j < held_c[:, None], own_ids, -1))
        held, used = torch.cat([held_p, held_c]), used + int(private.sum())
    table = torch.cat([table_p, table_c])
    mapped = torch.bincount(table[table >= 0], minlength=blocks)
    free = ids[used:]
    ring = torch.full((blocks,), -1, dtype=torch.int64)
    head = int(_between(0, blocks - 1, 1, cpu))
    ring[(head + torch.arange(len(free))) % blocks] = free
    state = torch.tensor([head, len(free), 0, 0])
    s["tables"], views = _flat([held, table, ring, state, (mapped - 1).clamp(min=0)])
    s["held"], s["table"], s["ring"], s["ring_state"], s["shares"] = views
    s["start"] = s["tables"].clone()
    none = torch.full((parents,), -1)
    s["parent"] = _i32(torch.cat([none, source]))
    s["lengths"] = _i32(torch.cat([lengths, length_c]))
    s["ended"] = _i32(torch.cat([lengths, torch.zeros(n, dtype=torch.int64)]))
    # where a batch is cut: anywhere in what a request has, every ninth ends
    total = torch.cat([lengths, grown])
    cut = (torch.rand(requests, generator=cpu) * (total + 1)).long().clamp(max=total)
    s["cut"] = _i32(torch.where(torch.arange(requests) % 9 == 8, 0, torch.where(cut % BLOCK == 0, total, cut)))
    s["pools"], s["generations"] = [], []
    for _ in range(case["layers"]):
        for width in (KV, INDEX):
            s["pools"].append(torch.randn((blocks * BLOCK, width), generator=gpu, device="cuda", dtype=torch.bfloat16))
        s["generations"].append(torch.randint(0, 5, (blocks * BLOCK,), generator=gpu, device="cuda"))


def _prompts(case, s, cpu, gpu):
    """Requests in order of the prompt that they continue; behind them one table row a prompt."""
    n, runs, heads = case["batch"], case["runs"], case["heads"]
    prompt = torch.arange(n) * runs // n
    tokens = _spread(case["prefix_low"], case["prefix_high"], runs)
    nodes = _spread(case["nodes_low"], case["nodes_high"], n)
    context = tokens[prompt] + _between(case["own_low"], case["own_high"], n, cpu) - 1
    whole, held = tokens // BLOCK, (context + nodes + BLOCK - 1) // BLOCK
    private = held - whole[prompt]
    blocks = runs * (case["prefix_high"] // BLOCK + 1) + n * ((case["own_high"] + case["nodes_high"]) // BLOCK + 2)
    stride = (case["prefix_high"] + case["own_high"] + case["nodes_high"]) // BLOCK + 1
    ids = torch.randperm(blocks, generator=cpu)
    j = torch.arange(stride)[None]
    at = torch.cumsum(whole, 0) - whole
    table_p = torch.where(j < whole[:, None], ids[torch.where(j < whole[:, None], at[:, None] + j, 0)], -1)
    first = int(whole.sum()) + torch.cumsum(private, 0) - private
    mine = (j >= whole[prompt][:, None]) & (j < held[:, None])
    table = torch.where(mine, ids[torch.where(mine, first[:, None] + j - whole[prompt][:, None], 0)], table_p[prompt])
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(nodes, 0)])
    masks = []
    for t in nodes.tolist():  # every node sees itself and what its parent sees
        words = [1]
        for i in range(1, t):
            words.append(words[int(_between(0, i - 1, 1, cpu))] | 1 << i)
        masks += words
    s.update(q=torch.randn((int(cu[-1]), heads, KV), generator=gpu, device="cuda").bfloat16(),
             pool=torch.randn((blocks * BLOCK, KV), generator=gpu, device="cuda", dtype=torch.bfloat16),
             table=_i32(torch.cat([table, table_p])), context=_i32(context), cu=_i32(cu),
             mask=torch.tensor(masks).cuda(), nodes=int(nodes.max()), prefix=_i32(tokens[prompt]),
             holder=_i32(n + prompt),
             sink=torch.randn((heads,), generator=gpu, device="cuda") if case["sink"] else None)
    starts = [int((prompt < r).sum()) for r in range(runs + 1)]
    s["runs"] = [(starts[r], starts[r + 1], int(cu[starts[r]]), int(cu[starts[r + 1]]), n + r, int(whole[r]))
                 for r in range(runs)]
    s["longest"] = case["own_high"] + case["nodes_high"] + BLOCK


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator("cuda").manual_seed(seed)
    s = dict(op=case["op"], status=torch.zeros(1, dtype=torch.int32, device="cuda"))  # the program's status word
    (_prompts if case["op"] == "prefix" else _pages)(case, s, cpu, gpu)
    return s


# ------------------------------------------------------------ the plain forms
def _listed_moves(where, source, target, rows, room):
    """The moves of the marked entries in their order, behind them entries of no rows."""
    rank = torch.where(where, torch.cumsum(where, 0) - 1, room)
    moves = torch.tensor([-1, -1, 0, 0], dtype=torch.int32, device=where.device).repeat(room + 1, 1)
    entry = torch.stack([source * BLOCK, target * BLOCK, rows, torch.zeros_like(rows)], 1).to(torch.int32)
    moves.index_copy_(0, rank, torch.where(where[:, None], entry, moves[room]))
    moves[room] = moves.new_tensor([-1, -1, 0, 0])
    return moves[:room], where.sum().to(torch.int32).view(1)


def _taken(s, where):
    """Free blocks from the ring's head for the marked requests, in their order."""
    state, size = s["ring_state"], s["ring"].numel()
    rank = torch.cumsum(where, 0) - where.long()
    return s["ring"].long()[(state[0].long() + rank) % size]


def _fork(s):
    table, held, lengths = s["table"], s["held"], s["lengths"].long()
    child, source = s["parent"] >= 0, s["parent"].long().clamp(min=0)
    whole, tail = lengths // BLOCK, lengths % BLOCK
    rows = table[source].long()
    j = torch.arange(table.shape[1], device=table.device)[None]
    shared = child[:, None] & (j < whole[:, None])
    s["shares"].scatter_add_(0, torch.where(shared, rows, 0).reshape(-1), shared.to(torch.int32).reshape(-1))
    copies = child & (tail > 0)
    fresh = _taken(s, copies)
    last = rows.gather(1, whole.clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    moves = _listed_moves(copies, last, fresh, tail, len(lengths))
    at_tail = copies[:, None] & (j == whole[:, None])
    table.copy_(torch.where(shared, rows, torch.where(at_tail, fresh[:, None], table.long())))
    held.copy_(torch.where(child, (lengths + BLOCK - 1) // BLOCK, held.long()))
    state = s["ring_state"]
    state[0] = (state[0] + copies.sum()) % s["ring"].numel()
    state[1] -= copies.sum()
    return moves


def _release(s, lengths):
    table, held, shares, ring, state = s["table"], s["held"].long(), s["shares"], s["ring"], s["ring_state"]
    lengths, size = lengths.long(), ring.numel()
    need, tail = (lengths + BLOCK - 1) // BLOCK, lengths % BLOCK
    j = torch.arange(table.shape[1], device=table.device)[None]
    dropped = (j >= need[:, None]) & (j < held[:, None])
    last = table.long().gather(1, (need - 1).clamp(min=0)[:, None])[:, 0]
    copies = (tail > 0) & (shares.long()[last.clamp(min=0)] > 0)
    fresh = _taken(s, copies)
    moves = _listed_moves(copies, last, fresh, tail, len(lengths))
    dropped |= copies[:, None] & (j == need[:, None] - 1)
    shares.scatter_add_(0, torch.where(dropped, table.long(), 0).reshape(-1), -dropped.to(torch.int32).reshape(-1))
    free = shares < 0
    place = (state[0].long() + state[1].long() + torch.cumsum(free, 0) - 1) % size
    wide = torch.cat([ring, ring.new_zeros(1)])
    wide.scatter_(0, torch.where(free, place, size), torch.arange(size, device=ring.device, dtype=torch.int32))
    ring.copy_(wide[:size])
    shares.clamp_(min=0)
    at_tail = copies[:, None] & (j == need[:, None] - 1)
    table.copy_(torch.where(at_tail, fresh[:, None], torch.where(dropped, -1, table.long())))
    state[0] = (state[0] + copies.sum()) % size
    state[1] += free.sum() - copies.sum()
    s["held"].copy_(need)
    return moves


def _compact(s):
    table, held, shares, ring, state = s["table"], s["held"], s["shares"], s["ring"], s["ring_state"]
    blocks, dev = ring.numel(), ring.device
    mapped = torch.arange(table.shape[1], device=dev)[None] < held[:, None]
    live = torch.zeros(blocks + 1, dtype=torch.bool, device=dev)
    live[torch.where(mapped, table.long(), blocks).reshape(-1)] = True
    live = live[:blocks]
    ids, used = torch.arange(blocks, device=dev), live.sum()
    hole, mover = ~live & (ids < used), live & (ids >= used)
    room = max(blocks // 2, 1)
    holes = torch.zeros(blocks + 1, dtype=torch.int64, device=dev)
    holes.scatter_(0, torch.where(hole, torch.cumsum(hole, 0) - 1, blocks), ids)
    target = torch.where(mover, holes[(torch.cumsum(mover, 0) - 1).clamp(min=0)], ids)
    moves = _listed_moves(mover, ids, target, torch.full_like(ids, BLOCK), room)
    table.copy_(torch.where(mapped, target[table.long().clamp(min=0)], table.long()))
    kept = torch.where(mover, 0, shares)
    shares.copy_(torch.where(hole, 0, kept).index_add(0, target, torch.where(mover, shares, 0)))
    ring.copy_(torch.where(ids < blocks - used, ids + used, -1))
    state[0], state[1] = 0, blocks - used
    return moves


def _copy(s, moves):
    moves = moves[0].long()
    r = torch.arange(BLOCK, device=moves.device)[None]
    valid = r < moves[:, 2:3]
    source, target = (moves[:, 0:1] + r)[valid], (moves[:, 1:2] + r)[valid]
    for pool in s["pools"]:
        pool[target] = pool[source]
    for g in s["generations"]:
        g[target] += 1


def _attend(scores, values):
    """(maximum, sum of the weights, weighted values) of scores [..., rows, keys]."""
    top = scores.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, 0.0, top)
    weights = scores.sub_(base).exp_()
    return top, weights.sum(-1, keepdim=True), torch.matmul(weights, values)


def _prefix(s):
    q, pool, heads = s["q"].float(), s["pool"], s["q"].shape[1]
    context, cu, most = s["context"].long(), s["cu"].long(), s["nodes"]
    # the shared rows, once for all requests of a prompt
    parts = []
    for _, _, n0, n1, row, whole in s["runs"]:
        rows = (s["table"][row, :whole].long()[:, None] * BLOCK + torch.arange(BLOCK, device=q.device)).reshape(-1)
        if not whole:
            parts.append((q.new_full((n1 - n0, heads, 1), -math.inf), q.new_zeros((n1 - n0, heads, 1)),
                          q.new_zeros((n1 - n0, heads, DV))))
            continue
        keys = pool[rows].float()
        top, total, out = _attend(torch.mm(q[n0:n1].reshape(-1, KV) * SCALE, keys.T), keys[:, :DV])
        parts.append(tuple(t.view(n1 - n0, heads, -1) for t in (top, total, out)))
    top1, total1, out1 = (torch.cat(t) for t in zip(*parts))
    # each request's own rows
    first = s["prefix"].long() // BLOCK * BLOCK
    position = first[:, None] + torch.arange(s["longest"], device=q.device)
    page = (position // BLOCK).clamp(max=s["table"].shape[1] - 1)
    rows = s["table"][:len(context)].long().gather(1, page) * BLOCK + position % BLOCK
    keys = pool[rows.clamp(min=0)].float()
    node = (cu[:-1, None] + torch.arange(most, device=q.device)).clamp(max=len(q) - 1)
    scores = torch.bmm(q[node].reshape(len(context), most * heads, KV) * SCALE, keys.transpose(1, 2))
    drafted = (position - context[:, None])[:, None]
    bit = (s["mask"][node][..., None] >> drafted.clamp(0, 63)) & 1
    seen = (drafted < 0) | ((drafted < (cu[1:] - cu[:-1])[:, None, None]) & (drafted < 64) & (bit == 1))
    scores.view(len(context), most, heads, -1).masked_fill_(~seen[:, :, None], -math.inf)
    own_parts = _attend(scores, keys[..., :DV])
    every = torch.arange(len(q), device=q.device)
    owner = torch.searchsorted(cu[1:], every, right=True)
    top2, total2, out2 = (t.view(len(context), most, heads, -1)[owner, every - cu[owner]] for t in own_parts)
    # both, and the sink
    top = torch.maximum(top1, top2)
    if s["sink"] is not None:
        top = torch.maximum(top, s["sink"][:, None])
    top = torch.where(top == -math.inf, 0.0, top)
    a, b = torch.exp(top1 - top), torch.exp(top2 - top)
    total = a * total1 + b * total2
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"][:, None] - top)
    return torch.where(total > 0, (a * out1 + b * out2) / total, 0.0).to(s["q"].dtype)


# ------------------------------------------------------------------ one pass
def run(s):
    if s["op"] == "prefix":
        if not own:
            return _prefix(s)
        import deepseekrpc_b200
        ops = deepseekrpc_b200.extension()
        return ops.prefix_mla_decode(s["q"], s["pool"], s["table"], s["context"], s["cu"], s["mask"], s["nodes"],
                                     s["prefix"], s["holder"], SCALE, sink=s["sink"], status=s["status"])[0]
    tables = [s[k] for k in ("held", "table", "ring", "ring_state", "shares")]
    if s["op"] != "fork":
        s["tables"].copy_(s["start"])  # the same batch again; a fork's children end, so it needs no such thing
    if own:
        import deepseekrpc_b200
        ops = deepseekrpc_b200.extension()
        if s["op"] == "fork":
            moves, count, _ = ops.paged_fork(s["parent"], s["lengths"], *tables, status=s["status"])
        elif s["op"] == "trim":
            moves, count, _ = ops.paged_release(s["cut"], *tables, status=s["status"])
        else:
            moves, count, _ = ops.paged_compact(*tables, status=s["status"])
        ops.paged_copy(s["pools"], s["generations"], moves, count, status=s["status"])
        if s["op"] == "fork":  # the children end
            ops.paged_release(s["ended"], *tables, status=s["status"])
    else:
        moves, count = done = dict(fork=_fork, compact=_compact).get(s["op"], lambda s: _release(s, s["cut"]))(s)
        _copy(s, done)
        if s["op"] == "fork":
            _release(s, s["ended"])
    return [moves, count, *tables, *s["pools"], *s["generations"]]


def work(case):
    """Each input read once, each output written once; the sizes that vary by seed at their mean."""
    if case["op"] == "prefix":
        n, runs, heads = case["batch"], case["runs"], case["heads"]
        nodes = (case["nodes_low"] + case["nodes_high"]) / 2
        shared = (case["prefix_low"] + case["prefix_high"]) / 2 // BLOCK * BLOCK
        mine = (case["own_low"] + case["own_high"]) / 2 + nodes + (BLOCK / 2 if case["prefix_high"] % BLOCK else 0)
        rows = n * nodes * heads
        return dict(bytes=(runs * shared + n * mine) * KV * 2 + rows * (KV + DV) * 2,
                    flops=rows * (shared + mine) * 2 * (KV + DV))
    parents, n = case["parents"], case["parents"] * case["children"]
    length, row = (case["low"] + case["high"]) / 2, (KV + INDEX) * 2 + 8
    share = 1 if case["low"] == case["high"] else 0.5
    entries = n * length * share / BLOCK
    if case["op"] == "fork":  # mapped and dropped again; half a block copied
        rows = n * (case["low"] % BLOCK if share == 1 else BLOCK / 2)
        return dict(bytes=entries * 24 + rows * case["layers"] * 2 * row, flops=0)
    if case["op"] == "trim":  # half of the entries dropped; a child whose cut is in what it shares copies half a block
        return dict(bytes=(entries + parents * length / BLOCK) / 2 * 8 + n * BLOCK / 2 * case["layers"] * 2 * row, flops=0)
    live = parents * (length / BLOCK + 0.5) + 2 * n
    moved = live * max(0.0, 1 - live / case["blocks"])
    return dict(bytes=(entries + parents * length / BLOCK) * 8 + case["blocks"] * 4 +
                moved * BLOCK * case["layers"] * 2 * row, flops=0)


# ------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    if case["op"] != "prefix":
        return None  # whole numbers, and rows as they were
    s = prepare(case, seed)
    cu, words, context = s["cu"].tolist(), s["mask"].tolist(), s["context"].tolist()
    lanes = torch.arange(BLOCK, device="cuda")
    outs = []
    for r0, r1, _, _, row, whole in s["runs"]:
        prompt = s["pool"][(s["table"][row, :whole].long()[:, None] * BLOCK + lanes).reshape(-1)].double()
        for b in range(r0, r1):
            drafts, at = cu[b + 1] - cu[b], cu[b]
            mine = s["table"][b, whole:(context[b] + drafts + BLOCK - 1) // BLOCK].long()
            rows = s["pool"][(mine[:, None] * BLOCK + lanes).reshape(-1)].double()
            past = context[b] - whole * BLOCK
            for t in range(drafts):
                branch = [past + i for i in range(drafts) if words[at + t] >> i & 1]
                kept = torch.cat([prompt, rows[:past], rows[branch]])
                e = (s["q"][at + t].double() @ kept.T) * SCALE
                if s["sink"] is not None:  # a logit of its own, whose value is zero
                    e = torch.cat([e, s["sink"].double()[:, None]], 1)
                    kept = torch.cat([kept, torch.zeros_like(kept[:1])])
                outs.append(torch.softmax(e, -1) @ kept[:, :DV])
    return torch.stack(outs)
