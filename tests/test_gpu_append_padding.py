"""Appends of batches of a fixed size whose last rows are padding: sequence and position -1,
as the block plan marks them.  All results are equal bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from deepseekrpc_b200 import _native, cuda_ops
from oracle import append_kv_index, paged_rows

pytestmark = pytest.mark.gpu


def batch(seq, positions, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    values = [torch.randn((len(seq), w), generator=gen, device="cuda").bfloat16() for w in (576, 128)]
    for v, s, p in zip(zip(*values), seq, positions):
        if s == p == -1:  # what stands in a padding row does not count
            v[0].fill_(float("nan")), v[1].fill_(float("inf"))
    return (torch.tensor(seq, dtype=torch.int32, device="cuda"), torch.tensor(positions, dtype=torch.int32, device="cuda"),
            *values)


CASES = [
    ([0, 1, -1, -1], [5, 70, -1, -1], 0),          # behind the last row
    ([-1, 0, -1, 0, 1], [-1, 5, -1, 6, 70], 0),    # anywhere
    ([-1, -1, -1], [-1, -1, -1], 0),               # nothing but padding
    ([0, -1, -1], [5, 5, -1], 3),                  # a sequence of -1 with a position is none
    ([0, 1, -1], [5, -1, -1], 3),                  # nor a position of -1 with a sequence
]


@pytest.mark.parametrize("ring", [False, True])
@pytest.mark.parametrize("seq,positions,code", CASES)
def test_padding_is_skipped(cuda, seq, positions, code, ring):
    pools = [torch.randn((4 * 64, w), device="cuda").bfloat16() for w in (576, 128)]
    swa = torch.randn((2, 128, 576), device="cuda").bfloat16() if ring else None
    table = np.array([[3, 0], [1, 2]], np.int32)
    generations = torch.randint(0, 9, (256,), device="cuda")
    s, p, kv, ix = batch(seq, positions, len(seq))
    rows = paged_rows(table, 4, seq, positions)
    expected = generations[torch.from_numpy(rows).cuda()]  # -1: the last row's, not looked at
    bits = lambda t: None if t is None else t.view(torch.int16).cpu().numpy().view(np.uint16)  # noqa: E731
    want = [bits(t) if t is None else bits(t).copy() for t in (*pools, swa)]
    gens = generations.cpu().numpy().copy()
    codes = append_kv_index(want[0], want[1], gens, rows, seq, positions, expected.cpu().numpy(), bits(kv), bits(ix),
                            want[2])
    status = cuda_ops.extension().append_kv_index(*pools, generations, torch.from_numpy(table).cuda(), s, p, expected, kv,
                                                  ix, swa)
    assert int(status.item()) == code and codes == ({code} if code else set())
    for got, ref in zip((*pools, swa), want):
        assert ref is None or np.array_equal(bits(got), ref)
    assert np.array_equal(generations.cpu().numpy(), gens)


def test_padding_is_skipped_in_ring_pools(cuda):
    p = _native.ptr
    pools = [torch.zeros((300, w), device="cuda").bfloat16() for w in (576, 128)]
    rings = [torch.tensor([[0, 100, 37], [100, 150, 3]], device="cuda"), torch.tensor([[150, 100, 0], [0, 150, 149]], device="cuda")]
    gens = [torch.zeros(300, dtype=torch.int64, device="cuda") for _ in range(2)]
    expected = torch.zeros(4, dtype=torch.int64, device="cuda")
    s, pos, kv, ix = batch([0, -1, 1, -1], [70, -1, 20, -1], 9)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    rc = _native.library().dsr_append_kv_index_ring(
        p(pools[0]), 300, p(rings[0]), p(gens[0]), p(expected), p(pools[1]), 300, p(rings[1]), p(gens[1]), p(expected), 2,
        p(s), p(pos), p(kv), p(ix), p(err), 4, _native.stream_handle())
    assert rc == 0 and int(err.item()) == 0
    for pool, values, gen, rows in zip(pools, (kv, ix), gens, ([7, 123], [220, 19])):
        want, count = torch.zeros_like(pool), torch.zeros_like(gen)
        want[rows], count[rows] = values[[0, 2]], 1
        assert torch.equal(pool, want) and torch.equal(gen, count)
