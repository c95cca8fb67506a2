"""Gradients of the checked rotation, against the formula's transpose in 64 bits.

Tolerance of one value as for the rotation itself: 2^-21 mscale (|g_a| + |g_b|), and
2^-8 of the value for a BF16 gradient.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops
from deepseekrpc_b200.rotary import rope_frequencies

pytestmark = pytest.mark.gpu
M = 1.25


def f64(t):
    return t.detach().double().cpu().numpy()


def expect(g, pos, freq, offset, interleaved, inverse):
    """(the transposed rotation of g, its tolerance)"""
    g3 = f64(g) if g.ndim == 3 else f64(g)[:, None]
    n = len(freq)
    i = np.arange(n)
    a, b = (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + i + n)
    ref = serving.rope(g3, pos.cpu().numpy(), f64(freq), offset, interleaved, M, not inverse)
    tol = np.zeros_like(g3)
    tol[..., a] = tol[..., b] = 2.0 ** -21 * M * (np.abs(g3[..., a]) + np.abs(g3[..., b]))
    if g.dtype == torch.bfloat16:
        tol += 2.0 ** -8 * (np.abs(ref) + tol)
    return ref.reshape(g.shape), tol.reshape(g.shape)


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_is_the_transposed_rotation(cuda, dtype, interleaved, inverse):
    gen = torch.Generator("cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    pos = torch.tensor([3, -1, 70001, 0, 12, 999, 4], dtype=torch.int32, device="cuda")  # -1: left as it is
    freq = rope_frequencies(16)[0].cuda()
    x = [rand(7, 3, 24).requires_grad_(), rand(7, 40).requires_grad_(), rand(7, 16)]
    out = cuda_ops.rope(x, pos, freq, offsets=[4, 24, 0], interleaved=[interleaved] * 3, mscale=M, inverse=inverse)
    assert [o.requires_grad for o in out] == [True, True, False]
    g = [rand(7, 3, 24), rand(7, 40)]
    torch.autograd.backward(out[:2], g)
    for t, grad, offset in zip(x, g, (4, 24)):
        ref, tol = expect(grad, pos, freq, offset, interleaved, inverse)
        assert t.grad.dtype == dtype and np.all(np.abs(f64(t.grad) - ref) <= tol)
    # the values are those of a call without gradients
    with torch.no_grad():
        plain = cuda_ops.rope(x, pos, freq, offsets=[4, 24, 0], interleaved=[interleaved] * 3, mscale=M, inverse=inverse)
    assert all(torch.equal(a, b) and not b.requires_grad for a, b in zip(out, plain))


def test_backward_of_broadcast_and_reordered_tensors(cuda):
    """One key for all heads; gradients that come expanded (a sum's) and with other strides;
    an output that nobody uses."""
    gen = torch.Generator("cuda").manual_seed(2)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    pos = torch.arange(5, dtype=torch.int32, device="cuda") * 37
    freq = rope_frequencies(8)[0].cuda()
    key, query = rand(5, 1, 12).requires_grad_(), rand(6, 5, 12).requires_grad_()
    heads, turned, unused = cuda_ops.rope([key.expand(5, 6, 12), query.transpose(0, 1), key], pos, freq,
                                          offsets=[4, 0, 0], interleaved=[True, False, True], mscale=M)
    w = rand(6, 12, 5)  # columns outermost: the gradient of `turned` has strided columns
    (heads.sum() + (turned.permute(1, 2, 0) * w).sum()).backward()
    ref, tol = expect(torch.ones(5, 6, 12, device="cuda"), pos, freq, 4, True, False)
    # six equal heads summed in 32 bits: five additions, each off by 2^-24 of at most the sum
    assert np.all(np.abs(f64(key.grad) - ref.sum(1, keepdims=True)) <= tol.sum(1, keepdims=True) +
                  5 * 2.0 ** -24 * np.abs(ref).sum(1, keepdims=True) * (1 + 2.0 ** -20))
    ref, tol = expect(w.permute(2, 0, 1).contiguous(), pos, freq, 0, False, False)
    assert np.all(np.abs(f64(query.grad) - ref.transpose(1, 0, 2)) <= tol.transpose(1, 0, 2))


def test_second_derivatives(cuda):
    """|R x|^2: gradient 2 R'R x, a second derivative along v of 2 R'R v."""
    gen = torch.Generator("cuda").manual_seed(3)
    x, v = (torch.randn((4, 2, 8), generator=gen, device="cuda") for _ in range(2))
    x.requires_grad_()
    pos = torch.tensor([1, 20, 300, 4000], dtype=torch.int32, device="cuda")
    args = dict(offsets=[0], interleaved=[True], mscale=M)
    y = cuda_ops.rope([x], pos, rope_frequencies(8)[0].cuda(), **args)[0]
    grad, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    second, = torch.autograd.grad((grad * v).sum(), x)
    # R'R = M^2 on the rotated columns (all of them).  R v is off by e = 2^-21 M 2 |v|; R' takes
    # an error of two values to at most sqrt(2) M e, and adds 2^-21 M (the sum of two values of
    # R v, of at most sqrt(2) M |v| each): in all 2^-21 M^2 |v| (2 sqrt(2) + 2 sqrt(2)) < 6 units
    size = float(v.abs().max()) * 2 * M * M
    assert torch.all((second - 2 * M * M * v).abs() <= 6 * 2.0 ** -21 * size + 2.0 ** -22 * size)


def test_raw_writes_into_tensors_with_history_are_refused(cuda):
    ext, freq = cuda_ops.extension(), rope_frequencies(8)[0].cuda()
    pos = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    w = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.randn(3, 8, device="cuda")
    y = x * w
    with pytest.raises(RuntimeError):
        ext.rope([y], [y], pos, freq, [0], [True])  # in place: y's own graph would not know
    with pytest.raises(RuntimeError):
        cuda_ops.rope([x], pos, freq, offsets=[0], interleaved=[True], out=[y])
    with pytest.raises(cuda_ops.ValidationError):
        cuda_ops.rope([x], pos, freq.clone().requires_grad_(), offsets=[0], interleaved=[True])
    with torch.no_grad():
        ext.rope([y], [y], pos, freq, [0], [True])
    # a tensor that autograd has saved is known to have changed
    z = x * w
    ext.rope([x], [x], pos, freq, [0], [True])
    with pytest.raises(RuntimeError):
        z.sum().backward()
    pool, q = torch.zeros(64, 576, device="cuda").bfloat16(), torch.zeros(1, 16, 576, device="cuda").bfloat16()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.zeros(1, 16, 512, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError):
        ext.tree_mla_decode(q, pool, i32(0)[None], i32(5), i32(0, 1), torch.ones(1, dtype=torch.int64, device="cuda"), 1,
                            0.1, out=out)
