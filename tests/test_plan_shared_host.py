"""The plan of a batch whose requests share blocks, without a GPU: refusals of the C ABI, and the
definition on a request that became shorter without giving its blocks back."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import serving
from deepseekrpc_b200 import _native

P = 256  # a pointer that passes the alignment checks; nothing is launched


@pytest.mark.parametrize("change", [dict(shares=None), dict(lengths=None), dict(batch=0), dict(tokens=-1)])
def test_host_side_validation_refuses_without_touching_a_device(change):
    lib = _native.library()
    a = dict(dict(lengths=P, shares=P, tokens=4, batch=2), **change)
    assert lib.dsr_paged_plan_shared(a["lengths"], P, P, P, 4, P, P, a["shares"], 8, P, P, P, a["tokens"], P, P, P,
                                     a["batch"], None) == _native.DSR_EINVAL
    assert _native.last_error()


@pytest.mark.parametrize("length,new,refused", [(320, 5, False), (300, 3, False), (192, 1, False), (191, 0, False),
                                                (191, 1, True), (150, 200, True), (128, 0, True), (0, 0, True)])
def test_definition_keeps_shared_blocks_from_the_ring_and_from_new_tokens(length, new, refused):
    table = np.array([[0, 1, 2, -1, -1, -1, -1], [0, 1, 2, 3, 4, -1, -1]], np.int32)
    ring = np.array([5, 6, 7, 8, 9, -1, -1, -1, -1, -1], np.int32)
    args = (np.array([192, length], np.int32), np.array([0, new], np.int32), np.array([3, 5], np.int32), table, ring,
            np.array([0, 5, 0, 0], np.int32), new)
    shares = np.array([1, 1, 1] + [0] * 7, np.int32)
    held, table, ring, state, maps, _, _, status = serving.paged_plan(*args, shares)
    assert status == refused and serving.paged_plan(*args)[-1] == 0
    if refused:
        assert np.array_equal(table, args[3]) and np.array_equal(ring, args[4]) and all((m == -1).all() for m in maps)
    else:
        free = [ring[(state[0] + i) % 10] for i in range(state[1])]
        assert not set(free) & {0, 1, 2} and not set(maps[2] // 64) & {0, 1, 2}
