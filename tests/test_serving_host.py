"""The operators around the decode path without a GPU: refusals of the C ABI, rotary
frequencies, and the 64-bit definitions the GPU tests rest on."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import _native, cuda_ops
from deepseekrpc_b200.rotary import rope_frequencies

P = 256  # a pointer that passes the alignment checks; nothing is launched


def plan(lib, lengths=P, held=P, table=P, stride=4, ring=P, state=P, blocks=8, seq=P, tokens=4, err=P, batch=2):
    return lib.dsr_paged_plan(lengths, P, held, table, stride, ring, state, blocks, seq, P, P, tokens, P, P, err, batch,
                              None)


def rope(lib, count=1, positions=P, pairs=4, mscale=1.0, tokens=2, **change):
    t = (_native.RopeTensor * max(count, 1))()
    for one in t:
        one.x, one.out, one.x_token, one.out_token = P, 4096, 8, 8
        one.heads, one.width, one.offset, one.interleaved, one.dtype = 1, 8, 0, 1, _native.DSR_F32
        for key, value in change.items():
            setattr(one, key, value)
    return lib.dsr_rope(t, count, positions, P, pairs, mscale, 0, P, tokens, None)


def sample(lib, logits=P, dtype=1, stride=100, vocab=100, temperature=P, tokens=P, rows=2):
    return lib.dsr_sample(logits, dtype, stride, vocab, temperature, P, P, P, P, tokens, P, P, rows, None)


def tree(lib, q=P, dtype=0, pool=P, blocks=8, table=P, stride=4, most=4, scale=1.0, out=P, out_dtype=0, ws=P,
         ws_bytes=1 << 40, batch=2, nodes=4, heads=16):
    return lib.dsr_tree_mla_decode(q, dtype, pool, blocks, table, stride, P, P, P, most, None, scale, out, out_dtype, None,
                                   ws, ws_bytes, P, batch, nodes, heads, None)


@pytest.mark.parametrize("call", [
    lambda n: plan(n, lengths=None), lambda n: plan(n, held=None), lambda n: plan(n, table=None),
    lambda n: plan(n, ring=None), lambda n: plan(n, state=None), lambda n: plan(n, seq=None), lambda n: plan(n, err=None),
    lambda n: plan(n, stride=0), lambda n: plan(n, stride=1 << 25), lambda n: plan(n, blocks=0),
    lambda n: plan(n, batch=0), lambda n: plan(n, batch=16385), lambda n: plan(n, tokens=-1),
    lambda n: plan(n, tokens=1 << 31),
    lambda n: rope(n, count=0), lambda n: rope(n, count=5), lambda n: rope(n, positions=None),
    lambda n: rope(n, pairs=0), lambda n: rope(n, pairs=257), lambda n: rope(n, mscale=0.0),
    lambda n: rope(n, mscale=math.inf), lambda n: rope(n, tokens=0), lambda n: rope(n, x=None),
    lambda n: rope(n, dtype=2), lambda n: rope(n, offset=1), lambda n: rope(n, offset=-1), lambda n: rope(n, heads=0),
    lambda n: rope(n, width=0), lambda n: rope(n, x=257), lambda n: rope(n, x=4096, out_token=9),
    lambda n: sample(n, logits=None), lambda n: sample(n, dtype=3), lambda n: sample(n, logits=257),
    lambda n: sample(n, vocab=0), lambda n: sample(n, vocab=262145), lambda n: sample(n, rows=0),
    lambda n: sample(n, rows=65536), lambda n: sample(n, stride=-1), lambda n: sample(n, temperature=None),
    lambda n: sample(n, tokens=None),
    lambda n: tree(n, q=None), lambda n: tree(n, dtype=2), lambda n: tree(n, out_dtype=-1), lambda n: tree(n, pool=None),
    lambda n: tree(n, table=None), lambda n: tree(n, stride=0), lambda n: tree(n, blocks=0), lambda n: tree(n, most=0),
    lambda n: tree(n, most=65), lambda n: tree(n, scale=0.0), lambda n: tree(n, scale=math.nan),
    lambda n: tree(n, out=None), lambda n: tree(n, out=264), lambda n: tree(n, ws=None), lambda n: tree(n, ws=128),
    lambda n: tree(n, ws_bytes=1000), lambda n: tree(n, batch=0), lambda n: tree(n, batch=65536),
    lambda n: tree(n, nodes=0), lambda n: tree(n, heads=24),
])
def test_host_side_validation_refuses_without_touching_a_device(call):
    lib = _native.library()
    assert call(lib) == _native.DSR_EINVAL
    assert _native.last_error()


def test_rope_tensor_matches_the_header():
    assert ctypes.sizeof(_native.RopeTensor) == 2 * 8 + 4 * 8 + 6 * 4


def test_tree_workspace_is_a_pure_host_function():
    lib = _native.library()
    assert lib.dsr_tree_mla_workspace_bytes(0, 16, 1) == 0
    assert lib.dsr_tree_mla_workspace_bytes(1, 64, 8) > lib.dsr_tree_mla_workspace_bytes(1, 16, 1) > 0


# ------------------------------------------------------------------ frequencies
def test_frequencies():
    plain, one = rope_frequencies(64)
    assert plain.dtype == torch.float64 and one == 1.0
    assert torch.allclose(plain, 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64), rtol=1e-15)
    assert torch.equal(rope_frequencies(64, scaling="linear", factor=8.0)[0], plain / 8)
    ntk = rope_frequencies(64, scaling="ntk", factor=8.0)[0]
    assert ntk[0] == 1 and abs(float(ntk[-1] / plain[-1]) * 8 - 1) < 1e-12
    yarn, m = rope_frequencies(64, scaling="yarn", factor=40.0)
    assert abs(m - (0.1 * math.log(40) + 1)) < 1e-15
    assert torch.equal(yarn[:8], plain[:8]) and torch.allclose(yarn[-8:], plain[-8:] / 40, rtol=1e-14)
    assert torch.all(yarn <= plain) and torch.all(yarn >= plain / 40 * (1 - 1e-14))
    same, m = rope_frequencies(64, scaling="yarn", factor=1.0)
    assert m == 1.0 and torch.allclose(same, plain, rtol=1e-15)
    for bad in (dict(dim=63), dict(dim=0), dict(dim=True), dict(dim=64, scaling="other"), dict(dim=64, base=1.0),
                dict(dim=64, factor=0.5), dict(dim=2, scaling="ntk", factor=2.0),
                dict(dim=64, scaling="yarn", beta_fast=1.0, beta_slow=2.0), dict(dim=64, factor=math.nan)):
        with pytest.raises(cuda_ops.ValidationError):
            rope_frequencies(**bad)


# ------------------------------------------------------------- the definitions
def test_plan_definition_keeps_every_block_once():
    rng = np.random.default_rng(1)
    batch, blocks, stride = 7, 60, 9
    lengths, held = np.zeros(batch, np.int32), np.zeros(batch, np.int32)
    table, ring = np.full((batch, stride), -1, np.int32), rng.permutation(blocks).astype(np.int32)
    state = np.array([13, blocks, 0, 0], np.int32)
    ring = np.roll(ring, 13)
    for _ in range(40):
        new = rng.integers(0, 150, batch).astype(np.int32)
        lengths[rng.random(batch) < 0.3] = 0
        new[lengths + new > stride * 64] = 0
        held, table, ring, state, maps, cu, visible, code = serving.paged_plan(lengths, new, held, table, ring, state,
                                                                               int(new.sum()) + 2)
        assert np.array_equal(held if code == 0 else visible, -(-visible // 64) if code == 0 else lengths)
        mapped = [table[b, j] for b in range(batch) for j in range(held[b])]
        free = [ring[(state[0] + i) % blocks] for i in range(state[1])]
        assert sorted(mapped + free) == list(range(blocks))
        if code == 0:
            lengths = (lengths + new).astype(np.int32)
            for s, p, slot in zip(*maps):
                assert (s == -1 and slot == -1) or slot == table[s, p // 64] * 64 + p % 64
            assert len(set(maps[2][maps[2] >= 0])) == int(new.sum()) == cu[-1]


@pytest.mark.parametrize("interleaved", [True, False])
def test_rope_definition_is_a_complex_product(interleaved):
    rng = np.random.default_rng(2)
    x, pos, freq = rng.standard_normal((5, 3, 20)), np.array([0, 7, -1, 100000, 3]), rng.random(6)
    y = serving.rope(x, pos, freq, 4, interleaved, 1.5)
    slab = x[..., 4:16]
    z = slab[..., 0::2] + 1j * slab[..., 1::2] if interleaved else slab[..., :6] + 1j * slab[..., 6:]
    z = z * 1.5 * np.exp(1j * pos[:, None, None] * freq)
    expect = x.copy()
    if interleaved:
        expect[..., 4:16:2], expect[..., 5:16:2] = z.real, z.imag
    else:
        expect[..., 4:10], expect[..., 10:16] = z.real, z.imag
    expect[2] = x[2]
    assert np.allclose(y, expect, atol=1e-10)
    back = serving.rope(y, pos, freq, 4, interleaved, 1 / 1.5, inverse=True)
    assert np.allclose(back, x, atol=1e-10)


def test_sample_definition_on_a_small_row():
    x = np.log(np.array([0.1, 0.4, 0.05, 0.25, 0.2]))  # order 1, 3, 4, 0, 2
    draw = lambda u, k=0, p=1.0, m=0.0, t=1.0: serving.sample(x, t, k, p, m, u)  # noqa: E731
    assert [draw(u)[0] for u in (0.0, 0.0999, 0.1001, 0.4999, 0.5001, 0.7, 0.9999)] == [0, 0, 1, 1, 2, 3, 4]
    assert draw(0.99, k=2) == (3, pytest.approx(0.25 / 0.65))
    assert draw(0.0, k=2) == (1, pytest.approx(0.4 / 0.65))
    assert draw(0.99, p=0.64)[0] == 3 and draw(0.99, p=0.66)[0] == 4  # 0.4 + 0.25 reach 0.64
    assert draw(0.99, k=2, p=0.6)[0] == 1  # of the 0.65 that the first two have
    assert draw(0.99, m=0.6)[0] == 3 and draw(0.0, m=0.7)[0] == 1
    assert draw(0.99, p=0.0)[0] == 1 and draw(0.5, t=0) == (1, 1.0)
    assert serving.sample(np.full(3, -np.inf), 1.0, 0, 1.0, 0.0, 0.5) == (-1, 0.0)


def test_tree_attention_definition_is_masked_softmax():
    rng = np.random.default_rng(3)
    nodes, heads, context = 4, 2, 6
    q, keys = rng.standard_normal((nodes, heads, 576)), rng.standard_normal((context + nodes, 576))
    masks, sink = [1, 3, 5, 0], rng.standard_normal(heads)
    for s in (sink, None):
        out, lse = serving.tree_attention(q, keys, context, masks, s, 0.05)
        logits = 0.05 * torch.einsum("nhd,kd->nhk", torch.from_numpy(q), torch.from_numpy(keys))
        hidden = torch.tensor([[j >= context and not masks[n] >> (j - context) & 1 for j in range(context + nodes)]
                               for n in range(nodes)])
        logits = logits.masked_fill(hidden[:, None], -math.inf)
        if s is not None:
            logits = torch.cat([logits, torch.from_numpy(s).expand(nodes, heads)[..., None]], -1)
        w = torch.softmax(logits, -1)[..., :context + nodes]
        assert np.allclose(out, (w @ torch.from_numpy(keys[:, :512])).numpy(), atol=1e-12)
        assert np.allclose(lse, torch.logsumexp(logits, -1).numpy(), atol=1e-12)
