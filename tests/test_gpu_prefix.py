"""Attention of requests that continue common prompts against the 64-bit formula, within
the tolerances of the tree attention (test_gpu_tree.py derives them: the parts of a row
are joined in FP32, by factors of relative error 2^-22 or so, far below the roundings
counted there)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_tree import SCALE, check, reference
from deepseekrpc_b200 import cuda_ops

pytestmark = pytest.mark.gpu


def problem(seed, prompts, heads, dtype=torch.bfloat16, tree="tree", sink=True, gap=0, kept=True):
    """prompts: (tokens, [(own tokens, nodes), ..]) each.  One table row per request, then one
    per prompt; kept: the requests' rows map the shared blocks too (else -1 stands there).
    What no request sees, and what is not mapped, holds NaN."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    contexts, nodes, prefix, holder = [], [], [], []
    n = sum(len(requests) for _, requests in prompts)
    for i, (tokens, requests) in enumerate(prompts):
        for mine, drafts in requests:
            contexts.append(tokens + mine)
            nodes.append(drafts)
            prefix.append(tokens)
            holder.append(n + i)
    contexts, nodes = np.asarray(contexts), np.asarray(nodes)
    shared = np.asarray(prefix) // 64
    held = -(-(contexts + nodes) // 64)
    stride = int(held.max()) + 2
    blocks = int((held - shared).sum() + sum(t // 64 for t, _ in prompts)) + 3
    ids = rng.permutation(blocks).astype(np.int32)
    table = np.full((n + len(prompts), stride), -1, np.int32)
    at = 0
    for i, (tokens, _) in enumerate(prompts):
        table[n + i, :tokens // 64] = ids[at:at + tokens // 64]
        at += tokens // 64
    pool = torch.full((blocks * 64, 576), float("nan"), device="cuda").bfloat16()
    rows = []
    for b in range(n):
        table[b, :shared[b]] = table[holder[b], :shared[b]]
        own = held[b] - shared[b]
        table[b, shared[b]:held[b]] = ids[at:at + own]
        at += own
        p = np.arange(contexts[b] + nodes[b])
        rows.append(torch.from_numpy(table[b, p // 64].astype(np.int64) * 64 + p % 64).cuda())
        if not kept:
            table[b, :shared[b]] = -1
    for i, (tokens, _) in enumerate(prompts):
        for block in table[n + i, :tokens // 64]:
            pool[block * 64:block * 64 + 64] = torch.randn((64, 576), generator=gen, device="cuda").bfloat16()
    for b in range(n):
        mine = rows[b][shared[b] * 64:]
        pool[mine] = torch.randn((len(mine), 576), generator=gen, device="cuda").bfloat16()
    masks = []
    for t in nodes:
        for i in range(t):
            if tree == "tree":  # itself and what its parent sees
                parent = masks[len(masks) - i + int(rng.integers(0, i))] if i else 0
                masks.append(parent | 1 << i)
            elif tree == "none":
                masks.append(0)
            else:  # anything, bits past the nodes too
                masks.append(int(rng.integers(0, 1 << 63)) * 2 + int(rng.integers(0, 2)))
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32).cuda()  # noqa: E731
    total = int(nodes.sum())
    d = dict(q=torch.randn((total + gap, heads, 576), generator=gen, device="cuda").to(dtype), pool=pool,
             table=torch.from_numpy(table).cuda(), context=i32(contexts), cu=i32(np.concatenate([[0], np.cumsum(nodes)])),
             mask=torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks] + [0] * gap, dtype=torch.int64).cuda(),
             sink=torch.randn(heads, generator=gen, device="cuda") if sink else None, most=int(max(nodes.max(), 1)),
             prefix=i32(prefix), holder=i32(holder))
    return d, rows, masks


def call(d, **more):
    return cuda_ops.extension().prefix_mla_decode(d["q"], d["pool"], d["table"], d["context"], d["cu"], d["mask"],
                                                  d["most"], d["prefix"], d["holder"], SCALE, sink=d["sink"], **more)


def verify(d, rows, masks, requests=None):
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    check(d, rows, masks, out, lse, requests)
    return out, lse


ONE = [(0, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sink", [True, False])
@pytest.mark.parametrize("heads,prompts", [
    (16, [(0, ONE)]), (16, [(63, ONE)]), (16, [(64, ONE)]), (16, [(64, [(0, 1), (1, 1)])]), (16, [(100, [(5, 1)] * 3)]),
    (32, [(128, [(0, 2)] * 5), (192, [(70, 1), (0, 3)])]), (64, [(1000, [(3, 1)] * 9)]),
    (128, [(320, [(0, 1), (64, 1), (63, 2)]), (0, [(10, 1)]), (129, [(200, 1)])]), (16, [(640, [(9, 1)] * 40)]),
    (128, [(2000, [(1, 1)] * 33)]), (64, [(700, [(5, 64), (0, 7)])]), (32, [(5, [(3, 1)] * 4)]),
])
def test_against_the_formula(cuda, dtype, sink, heads, prompts):
    verify(*problem(heads + len(prompts), prompts, heads, dtype, sink=sink))


@pytest.mark.parametrize("tree", ["none", "any"])
def test_masks_and_tables_without_the_shared_blocks(cuda, tree):
    """Nodes that see the prompt alone; arbitrary words.  Shared blocks are the holder's only."""
    d, rows, masks = problem(3, [(256, [(0, 3), (64, 5), (7, 0), (0, 64)]), (0, [(0, 2), (1, 1)])], 16, tree=tree,
                             sink=tree == "any", kept=False)
    out, lse = verify(d, rows, masks)
    if tree == "none":
        assert torch.all(out[72:74] == 0) and torch.all(torch.isneginf(lse[72:74]))


def test_ragged_runs(cuda):
    rng = np.random.default_rng(4)
    prompts = [(int(rng.integers(0, 3000)), [(int(rng.integers(0, 400)), int(rng.integers(0, 4)))
                                             for _ in range(rng.integers(1, 30))]) for _ in range(20)]
    for heads in (16, 128):
        verify(*problem(5, prompts, heads, tree="any"))


def test_long_prompts_split_over_the_gpu(cuda):
    verify(*problem(6, [(70001, [(33, 1)] * 6), (9000, [(20000, 2)])], 64), requests=[0, 5, 6])


def test_many_requests(cuda):
    """More runs than threads of the plan, and a run of many requests."""
    rng = np.random.default_rng(7)
    prompts = [(int(rng.integers(0, 200)), [(int(rng.integers(0, 5)), 1)] * int(rng.integers(1, 3))) for _ in range(1500)]
    d, rows, masks = problem(8, prompts + [(500, [(1, 1)] * 600)], 16)
    verify(d, rows, masks, requests=[0, 1, 2, 700, 1500, len(rows) - 600, len(rows) - 300, len(rows) - 1])


def test_the_largest_batch(cuda):
    d, rows, masks = problem(20, [(64, [(1, 1)] * 16384)], 16)
    verify(d, rows, masks, requests=[0, 1, 7, 8, 8191, 16383])
    d["context"][77] = -1
    out, status = call(d, out=torch.full((16384, 16, 512), 5.0, device="cuda"))
    assert int(status.item()) == 1 and torch.all(out[77] == 5.0)
    check(d, rows, masks, out, requests=[0, 76, 78, 16383])


def test_the_tree_attention_agrees(cuda):
    d, rows, masks = problem(9, [(1000, [(30, 2), (40, 3)] * 8), (64, ONE)], 32)
    out, status, lse = call(d, return_lse=True)
    table = d["table"][:len(rows)].contiguous()
    same = cuda_ops.extension().tree_mla_decode(d["q"], d["pool"], table, d["context"], d["cu"], d["mask"], d["most"],
                                                SCALE, sink=d["sink"], return_lse=True)
    assert int(status) == int(same[1]) == 0
    assert (out - same[0]).float().norm() <= 2 ** -7 * same[0].float().norm()
    assert torch.allclose(lse, same[2], rtol=0, atol=2 ** -10)


def test_many_places_for_few_requests(cuda):
    """Most of a batch is finished or not there: few rows, more than 32 requests."""
    for n in (31, 32, 33, 1025):
        requests = [(3, 0)] * n
        requests[n // 2] = requests[n - 1] = (70, 2)
        verify(*problem(n, [(500, requests)], 16), requests=[n // 2, n - 1])


@pytest.mark.parametrize("heads", [16, 64, 128])
def test_edges_of_tiles_and_groups(cuda, heads):
    """Own rows that end at, before and behind tiles of 128 that start at any block; drafts
    across them; groups of 128 rows that are nearly empty."""
    prompts = [(tokens, [(mine, drafts) for mine in (0, 1, 63, 64, 65, 127, 128, 129, 200) for drafts in (1, 5)])
               for tokens in (64, 128, 191, 320)]
    verify(*problem(heads, prompts, heads, tree="any"))


@pytest.mark.parametrize("heads,nodes", [(16, 3), (16, 5), (32, 3), (64, 3), (128, 2)])
def test_requests_across_groups_of_rows(cuda, heads, nodes):
    """Own rows, short and long, of requests whose rows lie in one group of 128 or across several."""
    mine = (1000, 10, 2000, 0, 5000, 513, 511, 127, 640, 641, 1, 4000)
    requests = [(m, (nodes, 1, 0, nodes + 4)[i % 4]) for i, m in enumerate(mine)]
    for prompts in ([(700, requests)], [(64, requests[:5]), (30, requests[5:]), (64, requests[::-1])]):
        verify(*problem(heads + nodes, prompts, heads, tree="any", kept=False))


def test_padding_queries_may_hold_anything(cuda):
    d, rows, masks = problem(17, [(700, [(3, 1)] * 10)], 32, gap=30)
    d["q"][10:] = float("nan")
    d["q"][20:] = float("inf")
    verify(d, rows, masks)


def test_scores_that_keep_growing(cuda):
    """Later keys score far higher: the running maximum moves and the output is rescaled."""
    d, rows, masks = problem(10, [(1400, [(20, 1)] * 5)], 32)
    q = d["q"].float()
    for b in range(5):
        direction = q[b, 0] / q[b, 0].norm()
        ramp = torch.linspace(-60, 60, len(rows[b]), device="cuda")[:, None]
        d["pool"][rows[b]] = (d["pool"][rows[b]].float() * (0.1 if b == 0 else 1) + ramp * direction / 2).bfloat16()
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    for b in range(5):
        # five such directions: G = sum |q k| SCALE log2(e) < 512, so E < 36 * 2^-23 * 512 < 2^-8
        ref, ref_lse, size = reference(d, rows, masks, b)
        got = out[b:b + 1].double().cpu().numpy()
        assert np.all(np.abs(got - ref) <= (2.0 ** -8 + 2.0 ** -8) * size * 1.01 + 2.0 ** -8 * np.abs(ref) + 1e-30)
        assert np.all(np.abs(lse[b:b + 1].double().cpu().numpy() - ref_lse) <= 2.0 ** -8 + 2.0 ** -14)


def test_rows_behind_the_last_request_and_output_buffer(cuda):
    d, rows, masks = problem(11, [(200, [(3, 2), (4, 3)])], 16, gap=4)
    out = torch.full((9, 16, 512), 7.0, device="cuda")
    res, status = call(d, out=out)
    assert int(status.item()) == 0 and res.data_ptr() == out.data_ptr()
    check(d, rows, masks, out)  # an FP32 output of a BF16 query
    assert torch.all(out[5:] == 7.0)
    fresh, _, lse = call(d, return_lse=True)
    assert torch.all(fresh[5:] == 0) and torch.all(torch.isneginf(lse[5:]))


def test_same_bits_again_and_on_another_stream_and_in_a_graph(cuda):
    d, rows, masks = problem(12, [(9000, [(50, 1)] * 9), (500, [(600, 6)])], 64)
    first = call(d)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call(d)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = call(d, status=status)[0]
    for step in range(3):
        d["context"][:9] = 9050 - 20 * step  # lengths and prompts are read at replay
        d["prefix"][:9] = 9000 - 3000 * step
        graph.replay()
        assert torch.equal(third, call(d)[0]) and int(status.item()) == 0
    d["context"][:9] = 9050
    graph.replay()
    check(d, rows, masks, third)


def test_bad_requests_are_reported(cuda):
    base, rows, masks = problem(13, [(200, [(5, 2), (0, 3), (70, 1)]), (64, [(0, 2)])], 16)
    for change in (dict(context=[205, -1, 270, 64]), dict(context=[205, 10 ** 6, 270, 64]),
                   dict(context=[205, 199, 270, 64]), dict(prefix=[200, -1, 200, 64]), dict(prefix=[200, 201, 200, 64]),
                   dict(holder=[4, -1, 4, 5]), dict(holder=[4, 6, 4, 5]), dict(cu=[0, 2, 1, 6, 8]),
                   dict(cu=[0, 2, 9, 6, 8])):
        d = dict(base)
        for key, value in change.items():
            d[key] = torch.tensor(value, dtype=torch.int32).cuda()
        out = torch.full((8, 16, 512), 5.0, device="cuda")
        _, status = call(d, out=out)
        assert int(status.item()) == 1
        check(base, rows, masks, out, requests=[0, 3])
        if "cu" not in change:
            check(base, rows, masks, out, requests=[2])
            assert torch.all(out[2:5] == 5.0)
    # sums that give all rows to both of two requests
    d = dict(base, cu=torch.tensor([0, 8, 0, 8, 8], dtype=torch.int32).cuda(), most=8)
    assert int(call(d)[1].item()) == 1
    for row, value in ((4, 10 ** 6), (4, -1), (0, -1)):  # a holder's block, a request's own
        d = dict(base, table=base["table"].clone())
        d["table"][row, 1 if row == 4 else 3] = value
        assert int(call(d)[1].item()) == 1
    with pytest.raises(cuda_ops.ValidationError):
        cuda_ops.prefix_mla_decode(d["q"], d["pool"], d["table"], d["context"], d["cu"], d["mask"], 2, d["prefix"],
                                   d["holder"], scale=SCALE)


def test_a_finished_request_among_others(cuda):
    """No nodes: its context, prefix and holder may be anything."""
    d, rows, masks = problem(14, [(200, [(5, 2), (0, 0), (70, 1)])], 16)
    for key, value in (("context", 0), ("prefix", 10 ** 6), ("holder", -5)):
        d[key][1] = value
        out, status = call(d)
        assert int(status) == 0
        check(d, rows, masks, out, requests=[0, 2])


def test_non_finite_values_are_reported(cuda):
    base, rows, masks = problem(15, [(300, [(5, 1)] * 12)], 16)
    for value in (float("nan"), float("inf")):
        for at in (150, 302):
            d = dict(base, pool=base["pool"].clone())
            d["pool"][rows[1][at], 5] = value
            assert int(call(d)[1].item()) == 2
        d = dict(base, q=base["q"].clone())
        d["q"][4, 15, 575] = value
        assert int(call(d)[1].item()) == 2
    d = dict(base, sink=base["sink"].clone())
    d["sink"][3] = float("inf")
    assert int(call(d)[1].item()) == 2


def test_refusals(cuda):
    d, _, _ = problem(16, [(100, [(5, 2)])], 16)
    names = ("q", "pool", "table", "context", "cu", "mask", "most", "prefix", "holder")
    ext = cuda_ops.extension()
    bad = [dict(q=d["q"].half()), dict(q=d["q"][:, :, :512]), dict(q=d["q"].transpose(0, 1)), dict(q=d["q"][:0]),
           dict(q=d["q"][:, :8].contiguous()), dict(pool=d["pool"].float()), dict(pool=d["pool"][:100]),
           dict(table=d["table"].long()), dict(table=d["table"][:, :0]), dict(table=d["table"][:0]),
           dict(context=d["context"].cpu()), dict(cu=d["cu"][:1]), dict(mask=d["mask"].int()), dict(mask=d["mask"][:1]),
           dict(prefix=d["prefix"].long()), dict(prefix=d["prefix"][:0]), dict(holder=d["holder"].float()),
           dict(holder=torch.cat([d["holder"]] * 2)), dict(most=0), dict(most=65)]
    for change in bad:
        with pytest.raises(RuntimeError):
            ext.prefix_mla_decode(*[{**d, **change}[k] for k in names], SCALE)
    args = [d[k] for k in names]
    for scale in (0.0, math.nan, -1.0):
        with pytest.raises(RuntimeError):
            ext.prefix_mla_decode(*args, scale)
        with pytest.raises(cuda_ops.ValidationError):
            cuda_ops.prefix_mla_decode(*args, scale=scale)
    with pytest.raises(RuntimeError):
        ext.prefix_mla_decode(*args, SCALE, sink=d["sink"][:3])
    with pytest.raises(RuntimeError):
        ext.prefix_mla_decode(*args, SCALE, out=torch.empty(2, 16, 576, device="cuda"))


def test_bad_requests_of_a_few_rows(cuda):
    """Up to 64 query rows: a refused request and the rows behind the last one stay as they are."""
    base, rows, masks = problem(18, [(200, [(5, 1), (0, 1)]), (64, ONE)], 16, gap=1)
    for change in (dict(context=[205, -1, 64]), dict(prefix=[200, 300, 64]), dict(holder=[3, 5, 4]), dict(cu=[0, 1, 0, 3])):
        d = dict(base)
        for key, value in change.items():
            d[key] = torch.tensor(value, dtype=torch.int32).cuda()
        out = torch.full((4, 16, 512), 5.0, device="cuda")
        _, status = call(d, out=out)
        assert int(status.item()) == 1
        check(base, rows, masks, out, requests=[0] if "cu" in change else [0, 2])
        if "cu" not in change:
            assert torch.all(out[1] == 5.0)
        assert torch.all(out[3] == 5.0)
    fresh, _, lse = call(base, return_lse=True)
    assert torch.all(fresh[3] == 0) and torch.all(torch.isneginf(lse[3]))


def test_a_bad_request_of_a_large_batch(cuda):
    """Its rows and those behind the last request stay as they are, the others are right."""
    d, rows, masks = problem(19, [(300, [(2, 1)] * 700), (0, [(9, 2)] * 500)], 16, gap=40)
    d["prefix"][700] = 10
    d["holder"][3] = -7
    out = torch.full((1740, 16, 512), 5.0, device="cuda")
    _, status = call(d, out=out)
    assert int(status.item()) == 1
    check(d, rows, masks, out, requests=[0, 2, 4, 699, 701, 1199])
    assert torch.all(out[3] == 5.0) and torch.all(out[700:702] == 5.0) and torch.all(out[1700:] == 5.0)
