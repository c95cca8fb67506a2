"""Generations that share entries are refused by the copies of rows, as one given twice is: two
threads would add to an entry at once."""
from __future__ import annotations

import pytest
import torch

from deepseekrpc_b200 import _native, cuda_ops
from test_sharing_host import copy


@pytest.mark.parametrize("gens", [(256, 256), (256, 264), (264, 256), (4096, 256, 256 + 8 * 63), (256 + 8 * 63, 256)])
def test_generations_that_overlap_are_refused(gens):
    lib = _native.library()
    assert copy(lib, gens=gens, rows=64, room=0) == _native.DSR_EINVAL
    assert "generations" in _native.last_error()


@pytest.mark.parametrize("gens", [(256, 256 + 8 * 64), (256 + 8 * 64, 256), (4096, 256, 256 + 8 * 64)])
def test_neighbouring_generations_are_not(gens):
    assert copy(_native.library(), gens=gens, rows=64, room=0) == _native.DSR_OK


@pytest.mark.gpu
def test_a_refused_copy_leaves_everything(cuda):
    store = torch.zeros(128 * 70 + 64, dtype=torch.int64, device="cuda")
    pool = torch.arange(128 * 8, device="cuda", dtype=torch.int16).view(128, 8)
    before = pool.clone()
    moves = torch.tensor([(0, 64, 5, 0)], dtype=torch.int32, device="cuda")
    count = torch.ones(1, dtype=torch.int32, device="cuda")
    apart = [store[128 * i:128 * i + 128] for i in range(70)]
    for bad in (apart[:3] + [store[64:192]], apart + [store[128 * 69 + 64:]]):  # in one launch, and over two
        version = pool._version
        with pytest.raises(RuntimeError):
            cuda_ops.extension().paged_copy([pool], bad, moves, count)
        assert torch.equal(pool, before) and pool._version == version and not store.any()
    assert int(cuda_ops.extension().paged_copy([pool], apart, moves, count)) == 0
    assert int(store.sum()) == 5 * 70 and torch.equal(pool[64:69], before[:5])
