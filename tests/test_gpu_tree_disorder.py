"""A refused request leaves the others' rows right, also where the node sums are in disorder and
the rows are joined from several parts.  Compared bit for bit with the same requests alone."""
from __future__ import annotations

import math

import pytest
import torch

from deepseekrpc_b200 import cuda_ops

pytestmark = pytest.mark.gpu


def attend(d, cu, rows, most):
    out = torch.full((len(d["q"]), 16, 512), 5.0, device="cuda")
    cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    _, status = cuda_ops.extension().tree_mla_decode(d["q"], d["pool"], d["table"][:len(cu) - 1], d["context"][:len(cu) - 1],
                                                     cu, d["mask"], most, 1 / math.sqrt(192), out=out)
    return out, int(status.item())


@pytest.mark.parametrize("more", [0, 40])  # with 40 further (empty) requests: the search of larger batches
def test_rows_of_good_requests_are_joined(cuda, more):
    gen = torch.Generator("cuda").manual_seed(more)
    n = 3 + more
    d = dict(q=torch.randn((8, 16, 576), generator=gen, device="cuda").bfloat16(),
             pool=torch.randn((64 * 24, 576), generator=gen, device="cuda").bfloat16(),
             table=torch.randperm(24, generator=gen, device="cuda").to(torch.int32).view(3, 8).repeat(1 + n // 3, 1)[:n].contiguous(),
             context=torch.full((n,), 500, dtype=torch.int32, device="cuda"),
             mask=torch.full((8,), 255, device="cuda"))
    # one unit a job in every call (few units), so that equal rows are cut alike
    ref, status = attend(d, [0, 5, 5, 5] + [5] * more, 5, 5)
    assert status == 0 and torch.all(ref[5:] == 5) and not torch.any((ref[:5] == 5).all(-1))
    # request 1 falls (refused), request 2 has too many nodes or the row 2 alone
    for cu, shared in (([0, 5, 2, 8], ()), ([0, 5, 2, 3], (2,))):
        out, status = attend(d, cu + [cu[-1]] * more, 8, 5)
        assert status == 1
        for row in range(5):
            if row not in shared:
                assert torch.equal(out[row], ref[row]), (cu, row)
        assert torch.all(out[5:] == 5)
