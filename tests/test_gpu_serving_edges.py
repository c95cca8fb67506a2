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
