"""Attention of drafted tokens on the GPU against the 64-bit formula.

Tolerances, for an output x = sum_i w_i v_i with weights w_i of sum at most 1.
Products of BF16 are exact in FP32; a score is accumulated in 36 steps of 16
products, each off by at most 2^-23 of what has been summed, which stays below
G = sum |q k| scale log2(e) < 64 for these inputs: 36 * 2^-23 * 64 < 2^-11 in log2
units, so a weight carries a relative error E < 2^-11 (exp's 2 ulp and the FP32 sums
are far below).  Each weight is then rounded to BF16, by at most 2^-8:
  |error| <= (2^-8 + 2^-11) sum_i w_i |v_i|  (+ 2^-8 |x| of a BF16 output).
The weights' roundings are independent, so over a node's outputs (values of random
sign, |x| ~ |w|_2 |v|) the error's 2-norm stays below 2^-7 of the output's: 2^-8 /
sqrt(3) from the weights, as much from the output, and a key too many or too few
among a thousand would exceed it.  The logarithm of the sum carries E and FP32's
rounding of numbers below 2^7: 2^-11 + 2^-17.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import _native, cuda_ops

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(192)


def problem(seed, contexts, nodes, heads, dtype=torch.bfloat16, tree="tree", sink=True, spare=3, gap=0):
    """A paged batch; unmapped rows and the rows past each request's end hold NaN."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    contexts, nodes = np.asarray(contexts), np.asarray(nodes)
    held = -(-(contexts + nodes) // 64)
    blocks = int(held.sum()) + spare
    ids = rng.permutation(blocks).astype(np.int32)
    table = np.full((len(contexts), int(held.max()) + 2), -1, np.int32)
    pool = torch.full((blocks * 64, 576), float("nan"), device="cuda").bfloat16()
    at, rows = 0, []
    for b, h in enumerate(held):
        table[b, :h] = ids[at:at + h]
        at += h
        p = np.arange(contexts[b] + nodes[b])
        rows.append(torch.from_numpy(table[b, p // 64].astype(np.int64) * 64 + p % 64).cuda())
        pool[rows[-1]] = torch.randn((len(p), 576), generator=gen, device="cuda").bfloat16()
    masks = []
    for t in nodes:
        for i in range(t):
            if tree == "tree":  # itself and what its parent sees
                parent = masks[len(masks) - i + int(rng.integers(0, i))] if i else 0
                masks.append(parent | 1 << i)
            elif tree == "chain":
                masks.append((2 << i) - 1)
            elif tree == "none":
                masks.append(0)
            else:  # anything, bits past the nodes too
                masks.append(int(rng.integers(0, 1 << 63)) * 2 + int(rng.integers(0, 2)))
    total = int(nodes.sum())
    d = dict(q=torch.randn((total + gap, heads, 576), generator=gen, device="cuda").to(dtype), pool=pool,
             table=torch.from_numpy(table).cuda(), context=torch.tensor(contexts, dtype=torch.int32).cuda(),
             cu=torch.tensor(np.concatenate([[0], np.cumsum(nodes)]), dtype=torch.int32).cuda(),
             mask=torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks] + [0] * gap, dtype=torch.int64).cuda(),
             sink=torch.randn(heads, generator=gen, device="cuda") if sink else None, most=int(max(nodes.max(), 1)))
    return d, rows, masks


def call(d, **more):
    return cuda_ops.extension().tree_mla_decode(d["q"], d["pool"], d["table"], d["context"], d["cu"], d["mask"],
                                                d["most"], SCALE, sink=d["sink"], **more)


def reference(d, rows, masks, b):
    n0, n1 = int(d["cu"][b]), int(d["cu"][b + 1])
    q = d["q"][n0:n1].bfloat16().double().cpu().numpy()
    keys = d["pool"][rows[b]].double().cpu().numpy()
    sink = None if d["sink"] is None else d["sink"].double().cpu().numpy()
    context = int(d["context"][b])
    ref, lse = serving.tree_attention(q, keys, context, masks[n0:n1], sink, SCALE)
    size = weighted_abs(q, keys, context, masks[n0:n1], sink)
    return ref, lse, size


def weighted_abs(q, keys, context, masks, sink):
    """sum_i w_i |v_i| of every output."""
    out = np.zeros((q.shape[0], q.shape[1], 512))
    for n in range(len(q)):
        seen = list(range(context)) + [context + j for j in range(len(q)) if int(masks[n]) >> j & 1]
        s = SCALE * (q[n] @ keys[seen].T)
        if sink is not None:
            s = np.concatenate([s, sink[:, None]], 1)
        if s.shape[1]:
            e = np.exp(s - s.max(1, keepdims=True))
            out[n] = (e / e.sum(1, keepdims=True))[:, :len(seen)] @ np.abs(keys[seen][:, :512])
    return out


def check(d, rows, masks, out, lse=None, requests=None):
    for b in range(len(rows)) if requests is None else requests:
        n0, n1 = int(d["cu"][b]), int(d["cu"][b + 1])
        if n0 == n1:
            continue
        ref, ref_lse, size = reference(d, rows, masks, b)
        got = out[n0:n1].double().cpu().numpy()
        tol = (2.0 ** -8 + 2.0 ** -11) * size + 1e-30
        if out.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
        assert np.all(np.isfinite(got)), b
        assert np.all(np.abs(got - ref) <= tol), (b, np.max(np.abs(got - ref) / tol))
        norms = np.linalg.norm((got - ref).reshape(n1 - n0, -1), axis=1), np.linalg.norm(ref.reshape(n1 - n0, -1), axis=1)
        assert np.all(norms[0] <= 2.0 ** -7 * norms[1]), (b, norms)
        if lse is not None:
            g = lse[n0:n1].double().cpu().numpy()
            assert np.array_equal(np.isneginf(g), np.isneginf(ref_lse))
            some = np.isfinite(ref_lse)
            assert np.all(np.abs(g[some] - ref_lse[some]) <= 2.0 ** -11 + 2.0 ** -17)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sink", [True, False])
@pytest.mark.parametrize("heads,contexts,nodes", [
    (16, [0], [1]), (16, [1], [1]), (16, [127], [1]), (16, [128], [2]), (16, [5000], [1]),
    (32, [63], [1]), (32, [64, 0, 700], [3, 1, 2]), (64, [65, 129], [1, 6]), (64, [3000], [8]),
    (128, [200], [1]), (128, [511, 0, 64], [2, 5, 1]), (16, [1000, 20], [64, 33]), (64, [300], [64]),
])
def test_against_the_formula(cuda, dtype, sink, heads, contexts, nodes):
    d, rows, masks = problem(heads + len(nodes), contexts, nodes, heads, dtype, sink=sink)
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0 and out.dtype == dtype
    check(d, rows, masks, out, lse)


@pytest.mark.parametrize("tree", ["chain", "none", "any"])
def test_masks(cuda, tree):
    """A chain; nodes that see only the context (or nothing at all); arbitrary words."""
    d, rows, masks = problem(3, [0, 200, 64, 1], [5, 9, 1, 64], 16, tree=tree, sink=tree == "any")
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    check(d, rows, masks, out, lse)
    if tree == "none":
        assert torch.all(out[:5] == 0) and torch.all(torch.isneginf(lse[:5]))


def test_ragged_batch_with_empty_requests(cuda):
    rng = np.random.default_rng(4)
    contexts, nodes = rng.integers(0, 1500, 300), rng.integers(0, 4, 300)
    contexts[7] = 20000
    nodes[7] = 3
    d, rows, masks = problem(5, contexts, nodes, 16, tree="any")
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    check(d, rows, masks, out, lse)


def test_long_context_split_over_the_gpu(cuda):
    d, rows, masks = problem(6, [70001, 33], [7, 2], 64)
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    check(d, rows, masks, out, lse)


def test_scores_that_keep_growing(cuda):
    """Later keys score far higher: the running maximum moves and the output is rescaled."""
    d, rows, masks = problem(7, [1200], [3], 32, sink=True)
    q = d["q"].float()
    direction = q[0, 0] / q[0, 0].norm()
    ramp = torch.linspace(-60, 60, 1203, device="cuda")[:, None]
    d["pool"][rows[0]] = (d["pool"][rows[0]].float() * 0.1 + ramp * direction).bfloat16()
    out, status, lse = call(d, return_lse=True)
    assert int(status.item()) == 0
    # here G reaches 60 |q| SCALE log2(e) < 256, so E < 36 * 2^-23 * 256 < 2^-9
    ref, ref_lse, size = reference(d, rows, masks, 0)
    got = out.double().cpu().numpy()
    assert np.all(np.abs(got - ref) <= (2.0 ** -8 + 2.0 ** -9) * size * 1.01 + 2.0 ** -8 * np.abs(ref) + 1e-30)
    assert np.all(np.abs(lse.double().cpu().numpy() - ref_lse) <= 2.0 ** -9 + 2.0 ** -15)


def test_rows_behind_the_last_request_and_output_buffer(cuda):
    d, rows, masks = problem(8, [100, 30], [2, 3], 16, gap=4)
    out = torch.full((9, 16, 512), 7.0, device="cuda")
    res, status = call(d, out=out)
    assert int(status.item()) == 0 and res.data_ptr() == out.data_ptr()
    check(d, rows, masks, out)  # an FP32 output of a BF16 query
    assert torch.all(out[5:] == 7.0)


def test_same_bits_again_and_on_another_stream_and_in_a_graph(cuda):
    d, rows, masks = problem(9, [9000, 500], [5, 6], 64)
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
        d["context"][0] = 9000 - 1000 * step  # lengths are read at replay
        graph.replay()
        assert torch.equal(third, call(d)[0]) and int(status.item()) == 0


def test_bad_requests_are_reported(cuda):
    base, rows, masks = problem(10, [100, 200, 64], [2, 3, 1], 16)
    for change in (dict(context=[100, -1, 64]), dict(context=[100, 10 ** 6, 64]), dict(cu=[0, 2, 1, 6]),
                   dict(cu=[0, 2, 5, 9])):
        d = dict(base)
        for key, value in change.items():
            d[key] = torch.tensor(value, dtype=torch.int32).cuda()
        out = torch.full((6, 16, 512), 5.0, device="cuda")
        _, status = call(d, out=out)
        assert int(status.item()) == 1
        check(base, rows, masks, out, requests=[0])
    d = dict(base, table=base["table"].clone())
    d["table"][1, 1] = 10 ** 6
    assert int(call(d)[1].item()) == 1
    d["table"][1, 1] = -1
    assert int(call(d)[1].item()) == 1
    d = dict(base, most=2)  # request 1 has three nodes
    out = torch.full((6, 16, 512), 5.0, device="cuda")
    assert int(call(d, out=out)[1].item()) == 1
    assert torch.all(out[2:5] == 5.0)
    with pytest.raises(cuda_ops.ValidationError):
        cuda_ops.tree_mla_decode(d["q"], d["pool"], d["table"], d["context"], d["cu"], d["mask"], 2, scale=SCALE)


def test_non_finite_values_are_reported(cuda):
    base, rows, masks = problem(11, [100, 200], [2, 3], 16)
    for value in (float("nan"), float("inf")):
        d = dict(base, pool=base["pool"].clone())
        d["pool"][rows[1][150], 5] = value
        _, status = call(d)
        assert int(status.item()) == 2
        d = dict(base, q=base["q"].clone())
        d["q"][4, 15, 575] = value
        _, status = call(d)
        assert int(status.item()) == 2
    d = dict(base, sink=base["sink"].clone())
    d["sink"][3] = float("inf")
    assert int(call(d)[1].item()) == 2


def test_refusals(cuda):
    d, _, _ = problem(12, [100], [2], 16)
    names = ("q", "pool", "table", "context", "cu", "mask")
    ext = cuda_ops.extension()
    bad = [dict(q=d["q"].half()), dict(q=d["q"][:, :, :512]), dict(q=d["q"].transpose(0, 1)), dict(q=d["q"][:0]),
           dict(q=d["q"][:, :8].contiguous()), dict(pool=d["pool"].float()), dict(pool=d["pool"][:100]),
           dict(table=d["table"].long()), dict(table=d["table"][:, :0]), dict(context=d["context"].cpu()),
           dict(cu=d["cu"][:1]), dict(mask=d["mask"].int()), dict(mask=d["mask"][:1])]
    for change in bad:
        args = [{**d, **change}[k] for k in names]
        with pytest.raises(RuntimeError):
            ext.tree_mla_decode(*args, 2, SCALE)
    args = [d[k] for k in names]
    for most, scale in ((0, SCALE), (65, SCALE), (2, 0.0), (2, float("nan"))):
        with pytest.raises(RuntimeError):
            ext.tree_mla_decode(*args, most, scale)
    with pytest.raises(RuntimeError):
        ext.tree_mla_decode(*args, 2, SCALE, sink=d["sink"][:3])
    with pytest.raises(RuntimeError):
        ext.tree_mla_decode(*args, 2, SCALE, out=torch.empty(2, 16, 576, device="cuda"))
    lib = _native.library()
    assert lib.dsr_tree_mla_workspace_bytes(1, 16, 1) > 0
