"""What the serving operators of a paged, tree-drafted decode step cost.

One such step: `paged_plan` gives every request the pool blocks that its new
tokens need and maps the tokens to pool rows, `rope` rotates the queries and
keys by their positions, `tree_mla_decode` attends from the drafted tokens of
each request over its cached rows and its own branch of the draft, and
`sample_logits` draws the next tokens.  `run` computes a case either with
elementary torch operations (own = False) or with this package's kernels.
"""
from __future__ import annotations

import math

import torch

own = False  # True: `run` calls this package's operators

BLOCK, KV, DV, INDEX, ROPE = 64, 576, 512, 128, 64
SCALE = 1 / math.sqrt(192)


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one request that decodes one token: latency alone
        dict(name="plan 1x1", op="plan", batch=1, low=4096, high=4096, new_low=1, new_high=1, stride=2048),
        # a decode batch with 8 drafted tokens each, contexts of 1 to 64K tokens
        dict(name="plan 256x8", op="plan", batch=256, low=1, high=65536, new_low=8, new_high=8, stride=1056),
        # admission of long prompts: 33 new requests, about a million tokens
        dict(name="plan admission", op="plan", batch=33, low=0, high=0, new_low=30000, new_high=34000, stride=2048),
        # the rotations of one decoded token: MLA query, index query, KV row and index key
        dict(name="rope 1 token", op="rope", tokens=1, heads=64, idx_heads=64, far=131072, inverse=False, query="f32"),
        # the gradient (inverse rotation) for an odd number of tokens of a batch
        dict(name="rope inverse 999", op="rope", tokens=999, heads=16, idx_heads=32, far=1048576, inverse=True,
             query="f32"),
        # a prefill chunk
        dict(name="rope prefill 8192", op="rope", tokens=8192, heads=128, idx_heads=64, far=65536, inverse=False,
             query="bf16"),
        # one sequence, plain decode of one token over a short cache
        dict(name="tree 1x1 4K", op="tree", batch=1, nodes_low=1, nodes_high=1, heads=16, low=4096, high=4096,
             sink=True),
        # one sequence, 8 drafted tokens over 128K cached ones
        dict(name="tree 1x8 128K", op="tree", batch=1, nodes_low=8, nodes_high=8, heads=64, low=131072, high=131072,
             sink=True),
        # a ragged batch: up to 6 drafted tokens each, contexts of 8K to 64K
        dict(name="tree 32x6 64K", op="tree", batch=32, nodes_low=3, nodes_high=6, heads=64, low=8192, high=65536,
             sink=False),
        # one row with the usual filters
        dict(name="sample 1", op="sample", rows=1, vocab=131072, dtype="f32", mode="usual"),
        # the rows of 8 requests with 6 drafted tokens each, nucleus alone
        dict(name="sample 48", op="sample", rows=48, vocab=131072, dtype="f32", mode="nucleus"),
        # a large batch of requests with their own settings, odd vocabulary
        dict(name="sample 511", op="sample", rows=511, vocab=128001, dtype="bf16", mode="mixed"),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(("plan", "rope", "tree", "sample"))
    if op == "plan":
        batch = _log(rng, 1, 512)
        high = _log(rng, 1, 65536)
        new = _log(rng, 1, max(1, min(32768, 1000000 // batch)))
        new_low = rng.choice((0, 1, new))
        return dict(op=op, batch=batch, low=rng.choice((0, high)), high=high, new_low=min(new_low, new), new_high=new,
                    stride=(high + new) // BLOCK + 1 + rng.randrange(9))
    if op == "rope":
        heads = rng.choice((16, 32, 64, 128))
        return dict(op=op, tokens=_log(rng, 1, 8192), heads=heads, idx_heads=rng.choice((16, 32, 64)),
                    far=_log(rng, 8, 1048576), inverse=rng.random() < 0.4, query=rng.choice(("f32", "bf16")))
    if op == "tree":
        while True:
            batch, nodes = _log(rng, 1, 32), rng.choice((1, rng.randint(2, 8), rng.randint(9, 64)))
            heads, high = rng.choice((16, 32, 64, 128)), _log(rng, 1, 131072)
            low = rng.choice((0, high, high // 8))
            # products and cached rows at most those of the largest listed case
            if batch * nodes * heads * high <= 32 * 6 * 64 * 36864 and batch * high <= 32 * 65536:
                return dict(op=op, batch=batch, nodes_low=rng.choice((1, nodes)), nodes_high=nodes, heads=heads,
                            low=low, high=high, sink=rng.random() < 0.5)
    vocab = _log(rng, 1000, 200000)
    return dict(op=op, rows=_log(rng, 1, min(1024, 511 * 128001 // vocab)), vocab=vocab,
                dtype=rng.choice(("f32", "bf16")), mode=rng.choice(("usual", "nucleus", "mixed", "plain")))


# ----------------------------------------------------------------- the inputs
def _between(low, high, n, gen):
    return torch.randint(low, high + 1, (n,), generator=gen, dtype=torch.int64)


def _spread(low, high, n):
    """Ragged counts that are the same for every seed: the outputs' shapes go by them."""
    return low + (torch.arange(n) * 1237 + high - low) % (high - low + 1)


def _i32(t):
    return t.to(torch.int32).cuda()


def _tables(held, stride, blocks, gen):
    """Block tables of `held` blocks each, and the ids that remain, in a seeded order."""
    ids = torch.randperm(blocks, generator=gen)
    at = torch.cumsum(held, 0) - held
    j = torch.arange(stride)[None]
    mapped = j < held[:, None]
    table = torch.where(mapped, ids[torch.where(mapped, at[:, None] + j, 0)], -1)
    return table, ids[int(held.sum()):]


def frequencies(pairs, base=10000.0, factor=40.0, original=4096, fast=32.0, slow=1.0):
    """Angular frequencies whose slow pairs are stretched by `factor` (interpolated
    between `fast` and `slow` turns over the original context), and the amplitude."""
    freq = base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    turns = lambda n: pairs * math.log(original / (n * 2 * math.pi)) / math.log(base)  # noqa: E731
    low, high = max(math.floor(turns(fast)), 0), min(math.ceil(turns(slow)), 2 * pairs - 1)
    ramp = ((torch.arange(pairs, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    gpu = torch.Generator("cuda").manual_seed(seed)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")  # the program's status word
    s = dict(op=case["op"], status=status)
    randn = lambda *shape: torch.randn(shape, generator=gpu, device="cuda")  # noqa: E731
    if case["op"] == "plan":
        n = case["batch"]
        lengths = _between(case["low"], case["high"], n, cpu)
        new = _spread(case["new_low"], case["new_high"], n)
        held = (lengths + BLOCK - 1) // BLOCK
        blocks = n * ((case["high"] + case["new_high"]) // BLOCK + 2)
        table, free = _tables(held, case["stride"], blocks, cpu)
        ring = torch.full((blocks,), -1, dtype=torch.int64)
        head = int(_between(0, blocks - 1, 1, cpu))
        ring[(head + torch.arange(len(free))) % blocks] = free
        s.update(lengths=_i32(lengths), new=_i32(new), none=_i32(torch.zeros(n)), held=_i32(held), table=_i32(table),
                 ring=_i32(ring), ring_state=_i32(torch.tensor([head, len(free), 0, 0])), tokens=int(new.sum()))
    elif case["op"] == "rope":
        n, heads = case["tokens"], case["heads"]
        kind = torch.float32 if case["query"] == "f32" else torch.bfloat16
        freq, mscale = frequencies(ROPE // 2)
        # the projections' outputs: query heads of 128 plain and 64 rotated columns, index
        # queries, latent rows and index keys; the rotated query columns go to the last 64
        # of the 576-wide absorbed query
        q = randn(n, heads, 128 + ROPE).to(kind)
        s.update(positions=_i32(_between(0, case["far"] - 1, n, cpu)), freq=freq.cuda(), mscale=mscale,
                 inverse=case["inverse"], offsets=[0, ROPE, DV, ROPE], interleaved=[True, False, True, False],
                 x=[q[..., 128:], randn(n, case["idx_heads"], INDEX).to(kind), randn(n, KV).bfloat16(),
                    randn(n, INDEX).bfloat16()])
        wide = torch.zeros((n, heads, KV), dtype=kind, device="cuda")
        s["out"] = [wide[..., DV:]] + [torch.empty_like(t) for t in s["x"][1:]]
    elif case["op"] == "tree":
        n, heads = case["batch"], case["heads"]
        context = _between(case["low"], case["high"], n, cpu)
        nodes = _spread(case["nodes_low"], case["nodes_high"], n)
        cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(nodes, 0)])
        held = (context + nodes + BLOCK - 1) // BLOCK
        table, _ = _tables(held, int(held.max()), int(held.sum()), cpu)
        masks = []
        for t in nodes.tolist():  # every node sees itself and what its parent sees
            words = [1]
            for i in range(1, t):
                words.append(words[int(_between(0, i - 1, 1, cpu))] | 1 << i)
            masks += [w - (1 << 64) if w >> 63 else w for w in words]
        s.update(q=randn(int(cu[-1]), heads, KV).bfloat16(), pool=randn(int(held.sum()) * BLOCK, KV).bfloat16(),
                 table=_i32(table), context=_i32(context), cu=_i32(cu), mask=torch.tensor(masks).cuda(),
                 sink=randn(heads) if case["sink"] else None, nodes=int(nodes.max()), longest=int((context + nodes).max()))
    else:
        n, vocab = case["rows"], case["vocab"]
        logits = randn(n, vocab) * 2.2
        likely = torch.rand((n, vocab), generator=gpu, device="cuda") < 40 / vocab
        logits += likely * 7 * torch.rand((n, vocab), generator=gpu, device="cuda")
        pick = lambda values: torch.tensor(values, device="cuda")[torch.randint(  # noqa: E731
            len(values), (n,), generator=gpu, device="cuda")]
        choices = dict(usual=((0.7,), (50,), (0.95,), (0.0,)), nucleus=((0.8, 1.0), (0,), (0.9, 0.95), (0.0,)),
                       plain=((1.0,), (0,), (1.0,), (0.0,)),
                       mixed=((0.0, 0.6, 0.8, 1.0, 1.3), (0, 1, 20, 50, 1000), (1.0, 0.95, 0.8), (0.0, 0.05)))
        temperature, top_k, top_p, min_p = (pick(v) for v in choices[case["mode"]])
        s.update(logits=logits if case["dtype"] == "f32" else logits.bfloat16(), temperature=temperature.float(),
                 top_k=top_k.to(torch.int32), top_p=top_p.float(), min_p=min_p.float(),
                 uniform=torch.rand((n,), generator=gpu, device="cuda"))
    return s


# ------------------------------------------------------------ the plain forms
def _plan(s, new, tokens):
    """Block counts to what the lengths need: blocks taken from the ring's head,
    blocks given back to its tail; then the map of the new tokens."""
    table, ring, state, held = s["table"], s["ring"], s["ring_state"], s["held"].long()
    total = (s["lengths"] + new).long()
    need = (total + BLOCK - 1) // BLOCK
    take, give = (need - held).clamp(min=0), (held - need).clamp(min=0)
    size, head, count = ring.numel(), state[0].long(), state[1].long()
    j = torch.arange(table.shape[1], device=table.device)[None]
    grows = (j >= held[:, None]) & (j < need[:, None])
    shrinks = (j >= need[:, None]) & (j < held[:, None])
    source = (head + (torch.cumsum(take, 0) - take)[:, None] + j - held[:, None]) % size
    target = (head + count + (torch.cumsum(give, 0) - give)[:, None] + j - need[:, None]) % size
    wide = torch.cat([ring, ring.new_zeros(1)])
    wide.scatter_(0, torch.where(shrinks, target, size).reshape(-1), table.reshape(-1))
    table.copy_(torch.where(grows, ring[torch.where(grows, source, 0)], torch.where(shrinks, -1, table)))
    ring.copy_(wide[:size])
    state[0] = (head + take.sum()) % size
    state[1] = count - take.sum() + give.sum()
    s["held"].copy_(need)
    ends = torch.cumsum(new, 0)
    cu = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    i = torch.arange(tokens, device=table.device)
    seq = torch.searchsorted(ends, i, right=True)
    position = s["lengths"].long()[seq] + i - cu.long()[seq]
    slot = table[seq, position // BLOCK] * BLOCK + position % BLOCK
    return [seq.to(torch.int32), position.to(torch.int32), slot.to(torch.int32), cu, total.to(torch.int32)]


def _rope(s, i):
    x, out, at = s["x"][i], s["out"][i], s["offsets"][i]
    angle = s["positions"].double()[:, None] * s["freq"]
    if x.dim() == 3:
        angle = angle[:, None]
    cos, sin = torch.cos(angle).float() * s["mscale"], torch.sin(angle).float() * s["mscale"]
    if s["inverse"]:
        sin = -sin
    r = x[..., at:at + ROPE].float()
    if s["interleaved"][i]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :ROPE // 2], r[..., ROPE // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    out.copy_(torch.cat([x[..., :at], r.to(x.dtype), x[..., at + ROPE:]], -1))
    return out


def _tree(s):
    q, heads = s["q"].float(), s["q"].shape[1]
    context, cu = s["context"].long(), s["cu"].long()
    batch, most = len(context), s["nodes"]
    position = torch.arange(s["longest"], device=q.device)
    rows = s["table"].long()[:, position // BLOCK] * BLOCK + position % BLOCK
    keys = s["pool"][rows.clamp(min=0)].float()  # [batch, longest, 576]
    slot = torch.arange(most, device=q.device)
    node = (cu[:-1, None] + slot).clamp(max=len(q) - 1)  # [batch, most]
    scores = torch.bmm(q[node].reshape(batch, most * heads, KV), keys.transpose(1, 2)) * SCALE
    drafted = (position - context[:, None])[:, None]  # [batch, 1, longest]
    bit = (s["mask"][node][..., None] >> drafted.clamp(0, 63)) & 1
    drafts = (cu[1:] - cu[:-1])[:, None, None]
    seen = (drafted < 0) | ((drafted < drafts) & (drafted < 64) & (bit == 1))
    scores = scores.view(batch, most, heads, -1).masked_fill_(~seen[:, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sink"] is not None:
        top = torch.maximum(top, s["sink"][:, None])
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"][:, None] - top)
    weights = torch.where(total > 0, weights / total, 0.0)
    out = torch.bmm(weights.view(batch, most * heads, -1), keys[..., :DV]).view(batch, most, heads, DV)
    every = torch.arange(len(q), device=q.device)
    owner = torch.searchsorted(cu[1:], every, right=True)
    return out[owner, every - cu[owner]].bfloat16()


def _sample(s):
    x, order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device=x.device)
    heat, k = s["temperature"][:, None], s["top_k"][:, None]
    weight = torch.exp((x.double() - x[:, :1].double()) / torch.where(heat > 0, heat, 1.0).double())
    keep = torch.where(heat > 0, (k <= 0) | (rank < k), rank == 0)
    before = torch.cumsum(weight * keep, -1)
    total = before[:, -1:].clone()
    before -= weight * keep
    p = s["top_p"][:, None].double()
    keep &= (rank == 0) | (p >= 1) | (before < p * total)
    keep &= weight >= s["min_p"][:, None].double()
    kept = torch.zeros_like(weight).scatter_(1, order, weight * keep)
    sums = torch.cumsum(kept, -1)
    token = (sums <= s["uniform"][:, None].double() * sums[:, -1:]).sum(-1, keepdim=True)
    chance = kept.gather(1, token) / sums[:, -1:]
    return [token[:, 0].to(torch.int32), chance[:, 0].float()]


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        import deepseekrpc_b200
        ops = deepseekrpc_b200.extension()
        if s["op"] == "plan":
            args = (s["held"], s["table"], s["ring"], s["ring_state"])
            grown = ops.paged_plan(s["lengths"], s["new"], *args, s["tokens"], status=s["status"])
            ops.paged_plan(s["lengths"], s["none"], *args, 0, status=s["status"])
            return grown[:5] + [s["held"], s["table"], s["ring"], s["ring_state"]]
        if s["op"] == "rope":
            ops.rope(s["x"], s["out"], s["positions"], s["freq"], s["offsets"], s["interleaved"], mscale=s["mscale"],
                     inverse=s["inverse"], status=s["status"])
            return s["out"]
        if s["op"] == "tree":
            return ops.tree_mla_decode(s["q"], s["pool"], s["table"], s["context"], s["cu"], s["mask"], s["nodes"],
                                       SCALE, sink=s["sink"], status=s["status"])[0]
        return ops.sample_logits(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniform"],
                                 status=s["status"])[:2]
    if s["op"] == "plan":
        # a step extends every request by its new tokens and, all drafts rejected, gives the blocks back
        grown = _plan(s, s["new"], s["tokens"])
        _plan(s, s["none"], 0)
        return grown + [s["held"], s["table"], s["ring"], s["ring_state"]]
    if s["op"] == "rope":
        return [_rope(s, i) for i in range(len(s["x"]))]
    return _tree(s) if s["op"] == "tree" else _sample(s)


def work(case):
    """Each input read once, each output written once; the sizes that vary by seed at their mean."""
    if case["op"] == "plan":
        n, length, new = case["batch"], (case["low"] + case["high"]) / 2, (case["new_low"] + case["new_high"]) / 2
        fresh = max(0.0, math.ceil((length + new) / BLOCK) - math.ceil(length / BLOCK))
        # two calls; the tokens' seq, position and slot; taken blocks move ring -> table -> ring
        return dict(bytes=n * (2 * 16 + 8) + n * new * 12 + n * fresh * 16, flops=0)
    if case["op"] == "rope":
        n, size = case["tokens"], 4 if case["query"] == "f32" else 2
        values = case["heads"] * ROPE * size + case["idx_heads"] * INDEX * size + (KV + INDEX) * 2
        return dict(bytes=n * (2 * values + 4), flops=n * ROPE * 3 * (case["heads"] + case["idx_heads"] + 2))
    if case["op"] == "tree":
        n, heads, length = case["batch"], case["heads"], (case["low"] + case["high"]) / 2
        nodes = (case["nodes_low"] + case["nodes_high"]) / 2
        return dict(bytes=n * ((length + nodes) * KV * 2 + nodes * heads * (KV + DV) * 2),
                    flops=n * nodes * heads * (length + nodes) * 2 * (KV + DV))
    return dict(bytes=case["rows"] * (case["vocab"] * (4 if case["dtype"] == "f32" else 2) + 28),
                flops=case["rows"] * case["vocab"] * 4)


# ------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None  # whole numbers
    if case["op"] == "rope":
        turn = torch.polar(torch.full((), s["mscale"], dtype=torch.float64, device="cuda"),
                           s["positions"].double()[:, None] * s["freq"] * (-1 if s["inverse"] else 1))
        outs = []
        for x, at, pairs_adjacent in zip(s["x"], s["offsets"], s["interleaved"]):
            y = x.double().clone()
            slab = y[..., at:at + ROPE]
            split = slab.unflatten(-1, (-1, 2) if pairs_adjacent else (2, -1))
            if not pairs_adjacent:
                split = split.transpose(-1, -2)
            z = torch.view_as_complex(split.contiguous()) * (turn if x.dim() == 2 else turn[:, None])
            z = torch.view_as_real(z)
            slab.copy_((z if pairs_adjacent else z.transpose(-1, -2)).flatten(-2))
            outs.append(y)
        return outs
    if case["op"] == "tree":
        outs = []
        cu, words = s["cu"].tolist(), s["mask"].tolist()
        for b, context in enumerate(s["context"].tolist()):
            at, drafts = cu[b], cu[b + 1] - cu[b]
            rows = (s["table"][b].long()[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).reshape(-1)
            keys = s["pool"][rows[:context + drafts]].double()
            for t in range(drafts):
                branch = [context + i for i in range(drafts) if words[at + t] >> i & 1]
                kept = torch.cat([keys[:context], keys[branch]])
                e = (s["q"][at + t].double() @ kept.T) * SCALE
                if s["sink"] is not None:  # a logit of its own, whose value is zero
                    e = torch.cat([e, s["sink"].double()[:, None]], 1)
                    kept = torch.cat([kept, torch.zeros_like(kept[:1])])
                outs.append(torch.softmax(e, -1) @ kept[:, :DV])
        return torch.stack(outs)
    tokens, chances = [], []
    every = s["logits"].double()
    settings = zip(s["temperature"].tolist(), s["top_k"].tolist(), s["top_p"].tolist(), s["min_p"].tolist(),
                   s["uniform"].tolist())
    for x, (heat, k, p, least, u) in zip(every, settings):
        if heat == 0:
            tokens.append((x == x.max()).nonzero()[0, 0])
            chances.append(torch.ones((), dtype=torch.float64, device="cuda"))
            continue
        chance = torch.softmax(x / heat, 0)
        ranked = torch.argsort(chance, descending=True, stable=True)
        ranked = ranked[:k] if k > 0 else ranked
        mass = chance[ranked] / chance[ranked].sum()
        if p < 1:
            ranked = ranked[:int((torch.cumsum(mass, 0) - mass < p).sum().clamp(min=1))]
        ranked = ranked[chance[ranked] >= least * chance.max()]
        left = ranked.sort().values
        ends = torch.cumsum(chance[left], 0)
        at = (ends / ends[-1] <= u).sum().clamp(max=len(left) - 1)
        tokens.append(left[at])
        chances.append(chance[left[at]] / ends[-1])
    return [torch.stack(tokens).to(torch.int32), torch.stack(chances)]
