"""Rotary positions on the GPU against the 64-bit formula.

Tolerance of one value: the cosine and sine are off by at most 2^-23 (sincospif,
2 ulp) + pi 2^-25 (the reduced angle rounded to 32 bits), their product with the
amplitude, the two products and the sum round by 2^-24 each: in all below
2^-21 mscale (|x_a| + |x_b|).  The angle itself is a product rounded to 64 bits, here
and (as two products) in the kernel: 4 * 2^-53 of the largest angle, which counts at
positions of 10^9.  A BF16 result rounds by 2^-8 of its value once more.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops
from deepseekrpc_b200.rotary import rope_frequencies

pytestmark = pytest.mark.gpu


def f64(t):
    return t.double().cpu().numpy()


def check(x, y, positions, freq, offset, interleaved, mscale, inverse, before=None):
    """y against the formula for x (2 or 3 dimensions); rows of position -1 equal `before`."""
    x3, y3 = (t[:, None] if t.ndim == 2 else t for t in (f64(x), f64(y)))
    pos, n = positions.cpu().numpy(), len(freq)
    ref = serving.rope(x3, pos, f64(freq), offset, interleaved, mscale, inverse)
    i = np.arange(n)
    a, b = (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + i + n)
    tol = np.zeros_like(x3)
    size = np.abs(x3[..., a]) + np.abs(x3[..., b])
    tol[..., a] = tol[..., b] = (2.0 ** -21 + 2.0 ** -51 * pos.max() * f64(freq).max()) * mscale * size
    if x.dtype == torch.bfloat16:
        rotated = np.concatenate([a, b])
        tol[..., rotated] += 2.0 ** -8 * (np.abs(ref[..., rotated]) + tol[..., rotated])
    real = pos >= 0
    assert np.all(np.abs(y3 - ref)[real] <= tol[real])
    if before is not None and (~real).any():
        b3 = f64(before)
        b3 = b3[:, None] if b3.ndim == 2 else b3
        assert np.array_equal(y3[~real], b3[~real])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,heads,width,offset,pairs,far", [
    (1, 1, 2, 0, 1, 10),              # the smallest
    (1, 64, 576, 512, 32, 131072),    # an MLA query
    (5, 3, 128, 64, 32, 1048576),     # an index query, far positions
    (3, 5, 27, 3, 7, 1000),           # off the 16-byte grid
    (2, 2, 512, 0, 256, 4096),        # the most pairs, whole head
    (1000, 16, 64, 0, 32, 2 ** 31 - 1),
    (301, 4, 80, 8, 20, 5000),        # half = 20: 16-byte pieces in fp32, not in bf16
])
def test_rotation(cuda, dtype, interleaved, tokens, heads, width, offset, pairs, far):
    gen = torch.Generator("cuda").manual_seed(tokens * 7 + pairs)
    x = torch.randn((tokens, heads, width), generator=gen, device="cuda").to(dtype)
    pos = torch.randint(0, far, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    pos[-1] = far - 1
    if tokens > 2:
        pos[1] = -1
    freq = rope_frequencies(2 * pairs)[0].cuda()
    for inverse, mscale in ((False, 1.0), (True, 1.37)):
        out = torch.full_like(x, 3.0)
        status = cuda_ops.extension().rope([x], [out], pos, freq, [offset], [interleaved], mscale=mscale,
                                           inverse=inverse)
        assert int(status.item()) == 0
        check(x, out, pos, freq, offset, interleaved, mscale, inverse, torch.full_like(x, 3.0))
        inplace = x.clone()
        cuda_ops.extension().rope([inplace], [inplace], pos, freq, [offset], [interleaved], mscale=mscale,
                                  inverse=inverse)
        real = pos >= 0
        assert torch.equal(inplace[real], out[real]) and torch.equal(inplace[~real], x[~real])


def test_four_strided_tensors_in_one_launch(cuda):
    """The tensors of a decode step: slabs of wider projections in, slabs of the absorbed query out."""
    n, gen = 37, torch.Generator("cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    proj, wide = rand(n, 16, 192), torch.full((n, 16, 576), 9.0, device="cuda")
    turned = rand(32, n, 128).transpose(0, 1)  # heads outside tokens
    kv, key = rand(n, 577).bfloat16()[:, 1:], rand(2 * n, 128).bfloat16()[::2]
    x = [proj[..., 128:], turned, kv, key]
    out = [wide[..., 512:], torch.zeros(n, 32, 128, device="cuda"), torch.zeros(n, 576, device="cuda").bfloat16(),
           torch.zeros(n, 128, device="cuda").bfloat16()]
    pos = torch.randint(0, 100000, (n,), generator=gen, device="cuda", dtype=torch.int32)
    freq, m = rope_frequencies(64, scaling="yarn", factor=40.0)
    offsets, inter = [0, 64, 512, 0], [True, False, True, False]
    status = cuda_ops.extension().rope(x, out, pos, freq.cuda(), offsets, inter, mscale=m)
    assert int(status.item()) == 0
    for a, b, o, i in zip(x, out, offsets, inter):
        check(a, b, pos, freq, o, i, m, False)
    assert torch.all(wide[..., :512] == 9.0)
    res = cuda_ops.rope(x, pos, freq.cuda(), offsets=offsets, interleaved=inter, mscale=m)
    assert all(torch.equal(a, b) for a, b in zip(res, out))


@pytest.mark.parametrize("interleaved", [True, False])
def test_gradient_is_the_inverse_rotation(cuda, interleaved):
    """<g, rope(x)> = <rope_inverse(g), x>, and against differences of the formula."""
    gen = torch.Generator("cuda").manual_seed(4)
    x, g = (torch.randn((9, 2, 24), generator=gen, device="cuda") for _ in range(2))
    pos = torch.arange(9, device="cuda", dtype=torch.int32) * 1001
    freq = rope_frequencies(16)[0].cuda()
    args = dict(offsets=[4], interleaved=[interleaved], mscale=1.25)
    grad = f64(cuda_ops.rope([g], pos, freq, inverse=True, **args)[0])
    x64, g64, h = f64(x), f64(g), 2.0 ** -10
    loss = lambda v: (g64 * serving.rope(v, pos.cpu().numpy(), f64(freq), 4, interleaved, 1.25)).sum()  # noqa: E731
    rng = np.random.default_rng(5)
    for _ in range(20):
        at = tuple(int(rng.integers(0, s)) for s in x64.shape)
        d = np.zeros_like(x64)
        d[at] = h
        # the map is linear: the difference is the derivative but for 64-bit rounding; the
        # kernel's own error as at the top, for a pair of |g| <= 5
        assert abs((loss(x64 + d) - loss(x64 - d)) / (2 * h) - grad[at]) <= 2.0 ** -21 * 1.25 * 10 + 1e-9
    y = f64(cuda_ops.rope([x], pos, freq, **args)[0])
    assert abs((g64 * y).sum() - (grad * x64).sum()) <= 2.0 ** -21 * 1.25 * 4 * np.abs(g64).sum() * np.abs(x64).max()


def test_bad_positions_and_padding(cuda):
    x = torch.randn(4, 8, device="cuda")
    pos = torch.tensor([3, -1, -2, 0], dtype=torch.int32, device="cuda")
    freq = rope_frequencies(8)[0].cuda()
    y = x.clone()
    status = cuda_ops.extension().rope([y], [y], pos, freq, [0], [True])
    assert int(status.item()) == 1
    assert torch.equal(y[1:3], x[1:3]) and torch.equal(y[3], x[3]) and not torch.equal(y[0], x[0])
    with pytest.raises(cuda_ops.ValidationError):
        cuda_ops.rope([x], pos, freq, offsets=[0], interleaved=[True])


def test_no_tokens(cuda):
    x = torch.empty(0, 8, device="cuda")
    pos = torch.empty(0, dtype=torch.int32, device="cuda")
    assert int(cuda_ops.extension().rope([x], [x], pos, rope_frequencies(8)[0].cuda(), [0], [True]).item()) == 0


def test_refusals(cuda):
    ext, freq = cuda_ops.extension(), rope_frequencies(8)[0].cuda()
    x, pos = torch.randn(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [
        ([x.half()], [x.half()], pos, freq, [0], [True]),            # type
        ([x], [x.bfloat16()], pos, freq, [0], [True]),               # out of another type
        ([x], [x], pos, freq, [1], [True]),                          # rotated columns outside the row
        ([x], [x], pos, freq, [-1], [True]),
        ([x], [x], pos, freq.float(), [0], [True]),                  # 32-bit frequencies
        ([x], [x], pos.long(), freq, [0], [True]),
        ([x], [x], pos[:3], freq, [0], [True]),                      # another number of tokens
        ([x.t()], [x.t()], torch.zeros(8, dtype=torch.int32, device="cuda"), freq[:2], [0], [True]),  # columns apart
        ([x] * 5, [x.clone() for _ in range(5)], pos, freq, [0] * 5, [True] * 5),
        ([], [], pos, freq, [], []),
        ([x], [x], pos, freq, [0, 0], [True]),
        ([x], [torch.as_strided(x, (4, 8), (0, 1))], pos, freq, [0], [True]),  # in place with other strides
    ]
    for args in bad:
        with pytest.raises(RuntimeError):
            ext.rope(*args)
    with pytest.raises(RuntimeError):
        ext.rope([x], [x], pos, freq, [0], [True], mscale=float("nan"))
