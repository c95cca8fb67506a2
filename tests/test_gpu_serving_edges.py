"""Calls at the edges of what the operators around the decode path allow.

Sampling: tokens equal, chances to 2^-24 relative plus 2^-40 (as one division of sums in
steps of 2^-44).  A weight (of at most 1) is rounded to a multiple of 2^-44, which is off by
2^-45 at most, and formed to 2^-42 of itself: a sum of n weights is off by n 2^-45 + 2^-42
times the sum.  Both sides of a comparison of the running sum with u times the total are
such sums, so another kept token is right where u times the total lies within twice that
of its share.  At u = 0 this always meets a first entry of less than 2^-45.  Plans: whole numbers, equal.  Attention: weights rounded to BF16
(2^-8), scores 2^-11 relative to the values' size, a BF16 output 2^-8; the norm 2^-7.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------------- sampling
def share(x, token, temperature, top_k, top_p, min_p):
    """(sum before, sum through, total, chance) of a token; it has to be kept."""
    weight = np.exp((x - x.max()) / temperature)
    order = np.lexsort((np.arange(len(x)), -x))
    if 0 < top_k < len(order):
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(weight[order])
        order = order[:max(1, int((mass - weight[order] < top_p * mass[-1]).sum()))]
    kept = np.sort(order[weight[order] >= min_p])
    assert token in kept
    low, total = weight[kept[kept < token]].sum(), weight[kept].sum()
    return low, low + weight[token], total, weight[token] / total


def sample(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniform=0.5):
    rows = len(logits)
    full = lambda v, t=torch.float32: torch.full((rows,), v, dtype=t, device="cuda")  # noqa: E731
    args = (full(temperature), full(top_k, torch.int32), full(top_p), full(min_p), full(uniform))
    tokens, chances, status = cuda_ops.extension().sample_logits(logits, *args)
    assert int(status.item()) == 0
    x = logits.double().cpu().numpy()
    for r in range(rows):
        token, chance = serving.sample(x[r], *(float(v[r]) if i != 1 else int(v[r]) for i, v in enumerate(args)))
        got = int(tokens[r])
        if got != token:
            d = [float(v[r]) for v in args]
            low, high, total, chance = share(x[r], got, d[0], int(d[1]), d[2], d[3])
            off = 2 * (len(x[r]) * 2.0 ** -45 + 2.0 ** -42 * total)
            assert low - off <= d[4] * total <= high + off, (r, got, token)
        assert abs(float(chances[r]) - chance) <= 2.0 ** -24 * chance + 2.0 ** -40, r


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,left,top_k", [(1000, 50, 200), (1800, 3, 1700), (2000, 150, 151), (1000, 50, 60)])
@pytest.mark.parametrize("temperature", [0.2, 1.0, 5.0])
def test_sampling_prefix_ends_among_entries_of_the_lowest_value(cuda, dtype, vocab, left, top_k, temperature):
    gen = torch.Generator("cuda").manual_seed(vocab + left)
    logits = torch.full((3, vocab), torch.finfo(dtype).min, dtype=dtype, device="cuda")
    at = torch.randperm(vocab, generator=gen, device="cuda")[:left]
    logits[:, at] = (torch.randn((3, left), generator=gen, device="cuda") * 2).to(dtype)
    for u in (0.0, 0.6, 0.99):
        sample(logits, temperature, top_k, uniform=u)
        sample(logits, temperature, top_k, top_p=0.9, uniform=u)


@pytest.mark.parametrize("temperature", [1e-31, 1e-32])
@pytest.mark.parametrize("top_k", [0, 150])
def test_sampling_of_tiny_values_at_a_tiny_temperature(cuda, temperature, top_k):
    """One step holds all: thousands of entries whose weight rounds to none."""
    gen = torch.Generator("cuda").manual_seed(9)
    x = -torch.rand((3, 40000), generator=gen, device="cuda", dtype=torch.float64) * 10 - 31.6
    x[:, ::1000] += 31.6  # 40 entries with weight; the others at 2^-45.6 to 2^-60
    logits = (x * temperature).float()
    for p in (0.5, 0.9, 1.0):
        sample(logits, temperature, top_k, p, uniform=0.7)


@pytest.mark.parametrize("temperature", [1e-30, 3e37, 3e38])
def test_sampling_extreme_temperatures(cuda, temperature):
    gen = torch.Generator("cuda").manual_seed(3)
    logits = torch.randn((2, 5000), generator=gen, device="cuda")
    sample(logits, temperature, 700, 0.8, uniform=0.3)
    logits = (torch.rand((2, 5000), generator=gen, device="cuda") * 2 - 1) * 3e38
    sample(logits, temperature, 700, 0.8, uniform=0.3)


def test_sampling_replays_with_other_values(cuda):
    logits = torch.randn((5, 20000), device="cuda")
    vec = [torch.full((5,), v, device="cuda") for v in (0.9, 0.95, 0.01, 0.4)]
    k = torch.full((5,), 50, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ext = cuda_ops.extension()
    call = lambda: ext.sample_logits(logits, vec[0], k, vec[1], vec[2], vec[3], status=status)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for top_k in (1, 50, 5000, 0):
        logits.copy_(torch.randn((5, 20000), device="cuda"))
        k.fill_(top_k)
        graph.replay()
        fresh = call()
        assert torch.equal(out[0], fresh[0]) and torch.equal(out[1], fresh[1])


# ------------------------------------------------------------------------ plan
def test_plan_reports_bad_blocks_that_are_given_back(cuda):
    args = [np.array([0, 10], np.int32), np.array([0, 1], np.int32), np.array([3, 1], np.int32),
            np.array([[4, 99, -5, -1], [2, -1, -1, -1]], np.int32), np.array([7, 6, 5, 0, 0, 0, 0, 0], np.int32),
            np.array([0, 3, 0, 0], np.int32)]
    expect = serving.paged_plan(*args, 1)
    d = [torch.from_numpy(a).cuda() for a in args]
    *_, status = cuda_ops.extension().paged_plan(*d, 1)
    assert int(status.item()) == expect[-1] == 1
    for got, want in zip(d[2:], expect[:4]):
        assert np.array_equal(got.cpu().numpy(), want)


def test_plan_writes_outputs_off_the_16_byte_grid(cuda):
    """The C call takes any int32 pointers: four tokens a store only where all three allow."""
    from deepseekrpc_b200 import _native
    p = _native.ptr
    lengths, new = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([5, 100], [70, 9]))
    held = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    table = torch.tensor([[3, -1, -1], [0, 1, -1]], dtype=torch.int32, device="cuda")
    ring = torch.tensor([2, 4, 5, 6, 7, 0, 0, 0], dtype=torch.int32, device="cuda")
    state = torch.tensor([0, 5, 0, 0], dtype=torch.int32, device="cuda")
    expect = serving.paged_plan(*(t.cpu().numpy() for t in (lengths, new, held, table, ring, state)), 83)
    store = torch.full((3, 100), -9, dtype=torch.int32, device="cuda")
    maps = [store[i, i + 1:i + 84] for i in range(3)]
    rest, err = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = _native.library().dsr_paged_plan(p(lengths), p(new), p(held), p(table), 3, p(ring), p(state), 8, p(maps[0]),
                                          p(maps[1]), p(maps[2]), 83, p(rest), p(rest[4:]), p(err), 2,
                                          _native.stream_handle())
    assert rc == 0 and int(err.item()) == 0
    for i in range(3):
        assert np.array_equal(maps[i].cpu().numpy(), expect[4][i])
        assert torch.all(store[i, :i + 1] == -9) and torch.all(store[i, i + 84:] == -9)


# ------------------------------------------------------------------ attention
def attend(lengths, counts, heads, seed, wide=False, padding=0, stream=None):
    """Requests of lengths (cached) and counts (drafted) with a page table in random order;
    NaN in every pool row that nobody sees and in the padding queries."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    batch, total = len(lengths), int(sum(counts))
    blocks = [-(-(c + n) // 64) for c, n in zip(lengths, counts)]
    ids = rng.permutation(sum(blocks) + 1)
    pool = torch.full(((sum(blocks) + 1) * 64, 576), float("nan"), device="cuda").bfloat16()
    table = np.full((batch, max(max(blocks), 1)), -1, np.int32)
    q = torch.randn((total + padding, heads, 576), generator=gen, device="cuda")
    q[total:] = float("nan")
    q = q if wide else q.bfloat16()
    sink = torch.randn(heads, generator=gen, device="cuda")
    masks, keys, at = [], [], 0
    for b in range(batch):
        table[b, :blocks[b]] = ids[at:at + blocks[b]]
        at += blocks[b]
        n = lengths[b] + counts[b]
        rows = torch.randn((n, 576), generator=gen, device="cuda").bfloat16()
        where = torch.from_numpy((table[b][np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64)).cuda()
        pool[where] = rows
        keys.append(rows.double().cpu().numpy())
        masks.append([int(rng.integers(0, 2 ** 62)) for _ in range(counts[b])])
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    scale = 1 / math.sqrt(192)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    words = torch.tensor([w for m in masks for w in m] + [0] * padding, dtype=torch.int64, device="cuda")
    call = [q, pool, torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"),
            torch.from_numpy(cu).cuda(), words, max(max(counts), 1), scale]
    out = torch.full((total + padding, heads, 512), 7.0, device="cuda")
    cuda_ops.extension().tree_mla_decode(*call, sink=sink, out=out, status=status)
    assert int(status.item()) == 0
    assert torch.all(out[total:] == 7)
    q64 = q.bfloat16().double().cpu().numpy()
    for b in range(batch):
        at = slice(cu[b], cu[b + 1])
        if counts[b] == 0:
            continue
        ref, _ = serving.tree_attention(q64[at], keys[b], lengths[b], masks[b], sink.double().cpu().numpy(), scale)
        got = out[at].double().cpu().numpy()
        size = np.abs(keys[b]).max()
        assert np.all(np.abs(got - ref) <= (2.0 ** -8 + 2.0 ** -11) * size), b
        assert np.linalg.norm(got - ref) <= 2.0 ** -7 * np.linalg.norm(ref) + 1e-30, b


@pytest.mark.parametrize("batch", [32, 33, 320, 321, 700])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_of_many_requests(cuda, batch, wide):
    rng = np.random.default_rng(batch)
    lengths = rng.integers(0, 300, batch).tolist()
    counts = rng.integers(0, 4, batch).tolist()
    lengths[batch // 2], counts[batch // 2] = 5000, 3
    attend(lengths, counts, 16, batch, wide, padding=5)


@pytest.mark.parametrize("nodes,heads", [(1, 32), (2, 16), (64, 16), (5, 128)])
def test_attention_of_long_contexts_in_each_group_size(cuda, nodes, heads):
    attend([20001, 64, 0], [nodes, nodes, max(nodes - 1, 1)], heads, nodes)


def test_attention_writes_nothing_where_no_request_has_nodes(cuda):
    out = torch.full((4, 16, 512), 3.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.zeros((4, 16, 576), device="cuda").bfloat16()
    pool = torch.zeros((128, 576), device="cuda").bfloat16()
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    mask = torch.zeros(4, dtype=torch.int64, device="cuda")
    for _ in range(3):
        cuda_ops.extension().tree_mla_decode(q, pool, table, none[:2] + 10, none, mask, 4, 0.1, out=out, status=status)
    assert int(status.item()) == 0 and torch.all(out == 3)
    # a bad request's status is there for the next operation on the stream
    bad = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    cuda_ops.extension().tree_mla_decode(q, pool, table, none[:2] - 5, bad, mask, 4, 0.1, out=out, status=status)
    seen = status.clone()
    assert int(seen.item()) == 1 and torch.all(out == 3)


def test_attention_on_two_streams_at_once(cuda):
    """Each call has its own workspace."""
    gen = torch.Generator("cuda").manual_seed(5)
    pool = torch.randn((8192, 576), generator=gen, device="cuda").bfloat16()
    table = torch.randperm(128, generator=gen, device="cuda").to(torch.int32)[None]
    context = torch.tensor([8100], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    mask = torch.full((8,), 255, dtype=torch.int64, device="cuda")
    qs = [torch.randn((8, 64, 576), generator=gen, device="cuda").bfloat16() for _ in range(2)]
    call = lambda q: cuda_ops.extension().tree_mla_decode(q, pool, table, context, cu, mask, 8, 0.07)[0]  # noqa: E731
    alone = [call(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        both = []
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                both.append(call(q))
        torch.cuda.synchronize()
        assert torch.equal(both[0], alone[0]) and torch.equal(both[1], alone[1])
