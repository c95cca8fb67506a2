"""Rotations whose outputs meet one another are refused before anything is launched."""
from __future__ import annotations

import pytest

from deepseekrpc_b200 import _native


def call(tokens=2, **second):
    t = (_native.RopeTensor * 2)()
    for i, one in enumerate(t):
        one.x, one.out = 4096 * (2 * i + 1), 4096 * (2 * i + 2)
        one.x_token = one.out_token = 16
        one.x_head = one.out_head = 8
        one.heads, one.width, one.offset, one.interleaved, one.dtype = 2, 8, 0, 1, _native.DSR_F32
    for key, value in second.items():
        setattr(t[1], key, value)
    return _native.library().dsr_rope(t, 2, 256, 256, 4, 1.0, 0, 256, tokens, None)


@pytest.mark.parametrize("second", [
    dict(x=8192, out=8192),               # in place on the other's output
    dict(out=8192),                       # the same output twice
    dict(out=4096),                       # the other's input
    dict(out_head=0), dict(out_token=0),  # a broadcast output
])
def test_overlapping_outputs_are_refused(second):
    assert call(**second) == _native.DSR_EINVAL
    assert "output" in _native.last_error()
