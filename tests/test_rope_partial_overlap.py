"""Rotations whose outputs meet other tensors away from their first element are refused
before anything is launched; views of one buffer that share no element are not."""
from __future__ import annotations

import pytest
import torch

from deepseekrpc_b200 import _native, cuda_ops
from deepseekrpc_b200.rotary import rope_frequencies

BASE = 1 << 20


def call(tensors, tokens=5, pairs=4):
    """tensors: (x, out, x_token, x_head, out_token, out_head, heads, width, offset[, dtype]),
    places in FP32 elements from BASE."""
    t = (_native.RopeTensor * len(tensors))()
    for one, (x, out, xt, xh, ot, oh, heads, width, offset, *dtype) in zip(t, tensors):
        one.x, one.out = BASE + 4 * x, BASE + 4 * out
        one.x_token, one.x_head, one.out_token, one.out_head = xt, xh, ot, oh
        one.heads, one.width, one.offset, one.interleaved = heads, width, offset, 1
        one.dtype = dtype[0] if dtype else _native.DSR_F32
    return _native.library().dsr_rope(t, len(tensors), 256, 256, pairs, 1.0, 0, 256, tokens, None)


FAR = 1 << 16


@pytest.mark.parametrize("tensors", [
    # one tensor: the output a token, a column, half a head after its input
    [(0, 16, 16, 8, 16, 8, 2, 8, 0)],
    [(0, 1, 100, 10, 100, 10, 2, 8, 0)],
    [(0, 4, 16, 8, 16, 8, 2, 8, 0)],
    # the output reversed over its input
    [(0, 64, 16, 8, -16, 8, 2, 8, 0)],
    # rows of the output that overlap: tokens, heads, heads of one token with the next's
    [(FAR, 0, 16, 8, 7, 8, 1, 8, 0)],
    [(FAR, 0, 16, 8, 16, 4, 2, 8, 0)],
    [(FAR, 0, 32, 8, 20, 8, 3, 8, 0)],
    # in place, rows that overlap within the rotated columns
    [(0, 0, 4, 0, 4, 0, 1, 8, 0)],
    # an output inside another tensor's output, or input; in place beside in place
    [(FAR, 0, 40, 0, 40, 0, 1, 12, 0), (2 * FAR, 8, 40, 0, 40, 0, 1, 12, 0)],
    [(FAR, 0, 40, 0, 40, 0, 1, 12, 0), (8, 2 * FAR, 40, 0, 40, 0, 1, 12, 0)],
    [(0, 0, 40, 0, 40, 0, 1, 12, 0), (6, 6, 40, 0, 40, 0, 1, 12, 0)],
    # shifted by tokens, its base outside the first one's rows
    [(FAR, 120, 40, 0, 40, 0, 1, 12, 0), (2 * FAR, 8, 40, 0, 40, 0, 1, 12, 0)],
    # heads inside tokens against tokens inside heads
    [(FAR, 0, 16, 8, 16, 8, 2, 8, 0), (2 * FAR, 0 + 8, 8, 40, 8, 40, 2, 8, 0)],
    # other element types: 8 BF16 columns are 4 places
    [(FAR, 0, 40, 0, 40, 0, 1, 12, 0), (2 * FAR, 11, 80, 0, 80, 0, 1, 8, 0, _native.DSR_BF16)],
])
def test_partial_overlaps_are_refused(tensors):
    assert call(tensors) == _native.DSR_EINVAL
    assert "output" in _native.last_error()


@pytest.mark.gpu
def test_slabs_of_one_projection_are_rotated(cuda):
    """Query, index query, row and key side by side in one buffer, in place and into the
    other half of it: the same values as apart."""
    gen = torch.Generator("cuda").manual_seed(1)
    n, freq = 33, rope_frequencies(64)[0].cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda") * 100
    wide = torch.randn((n, 2, 16 * 192 + 8 * 128 + 576 + 128), generator=gen, device="cuda")

    def slabs(t):
        q, i, kv, key = t.split([16 * 192, 8 * 128, 576, 128], -1)
        return [q.unflatten(-1, (16, 192)), i.unflatten(-1, (8, 128)), kv, key]

    args = ([128, 64, 512, 0], [True, False, True, False])
    apart = [t.clone() for t in slabs(wide[:, 0])]
    cuda_ops.extension().rope(apart, apart, pos, freq, *args)
    before = wide.clone()
    cuda_ops.extension().rope(slabs(wide[:, 0]), slabs(wide[:, 1]), pos, freq, *args)
    assert torch.equal(wide[:, 0], before[:, 0])
    assert all(torch.equal(a, b) for a, b in zip(slabs(wide[:, 1]), apart))
    cuda_ops.extension().rope(slabs(wide[:, 0]), slabs(wide[:, 0]), pos, freq, *args)
    assert all(torch.equal(a, b) for a, b in zip(slabs(wide[:, 0]), apart))


@pytest.mark.gpu
def test_views_between_one_another_are_rotated(cuda):
    """Even and odd tokens, the two parts of every head, heads outside tokens, a row read by
    all heads."""
    gen = torch.Generator("cuda").manual_seed(2)
    x = torch.randn((10, 6, 24), generator=gen, device="cuda")
    pos, freq = torch.arange(5, dtype=torch.int32, device="cuda"), rope_frequencies(8)[0].cuda()
    ext = cuda_ops.extension()
    for views in (lambda t: [t[::2], t[1::2]], lambda t: [t[:5, :, :12], t[:5, :, 12:]],
                  lambda t: [t[:5, ::2], t[:5, 1::2], t[5:]],
                  lambda t: [t.view(6, 10, 24).transpose(0, 1)[:5], t.view(6, 10, 24).transpose(0, 1)[5:]]):
        mine, apart = x.clone(), [v.clone() for v in views(x)]
        k = len(apart)
        ext.rope(views(mine), views(mine), pos, freq, [4] * k, [True] * k)
        ext.rope(apart, apart, pos, freq, [4] * k, [True] * k)
        assert all(torch.equal(a, b) for a, b in zip(views(mine), apart))
    one = x[:5, :1].expand(5, 6, 24)
    out = torch.empty(5, 6, 24, device="cuda")
    ext.rope([one], [out], pos, freq, [4], [True])
    apart = one.clone()
    ext.rope([apart], [apart], pos, freq, [4], [True])
    assert torch.equal(out, apart)
