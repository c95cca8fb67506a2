"""Sampling on the GPU against the 64-bit definition: tokens equal, chances to 32 bits.

A token can only differ when a uniform number or a filter's border falls within
the two computations' rounding (about 2^-44 of the mass): below 10^-6 over all
rows of this file.  A chance is one division of sums that carry 2^-44 steps,
rounded to 32 bits: 2^-24 relative, plus 2^-40 of steps for the smallest weights.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops

pytestmark = pytest.mark.gpu


def run(logits, **settings):
    rows = logits.shape[0]
    d = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniform=0.5)
    d.update(settings)
    kinds = dict(top_k=torch.int32)
    vec = {k: torch.as_tensor(np.broadcast_to(np.asarray(v), (rows,)).copy()).to(kinds.get(k, torch.float32)).cuda()
           for k, v in d.items()}
    tokens, chances, status = cuda_ops.extension().sample_logits(logits, **vec)
    return tokens.cpu().numpy(), chances.cpu().numpy(), int(status.item()), {k: v.cpu().numpy() for k, v in vec.items()}


def check(logits, **settings):
    tokens, chances, status, d = run(logits, **settings)
    assert status == 0
    x = logits.double().cpu().numpy()
    for r in range(len(x)):
        token, chance = serving.sample(x[r], *(d[k][r] for k in ("temperature", "top_k", "top_p", "min_p", "uniform")))
        assert tokens[r] == token, (r, tokens[r], token)
        assert abs(chances[r] - chance) <= 2.0 ** -24 * chance + 2.0 ** -40, r
    return tokens


def draw(seed, rows, vocab, spread=2.5):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randn((rows, vocab), generator=gen, device="cuda") * spread


SETTINGS = [
    dict(),
    dict(top_k=1), dict(top_k=7), dict(top_k=700), dict(top_k=10 ** 6),
    dict(top_p=0.9), dict(top_p=0.0), dict(top_p=0.999), dict(top_k=50, top_p=0.95),
    dict(min_p=0.05), dict(min_p=1.0), dict(top_k=3000, top_p=0.6, min_p=0.01),
    dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=50.0, top_p=0.5), dict(temperature=0.3, top_k=40),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 2), (3, 31), (5, 1000), (17, 4097), (2, 128001), (3, 262144)])
def test_filters(cuda, dtype, rows, vocab):
    logits = draw(vocab, rows, vocab).to(dtype)
    rng = np.random.default_rng(vocab)
    for settings in SETTINGS:
        check(logits, uniform=rng.random(rows).astype(np.float32) * np.float32(1 - 2.0 ** -24), **settings)


@pytest.mark.parametrize("rows", [40, 301])
def test_rows_with_their_own_settings(cuda, rows):
    rng = np.random.default_rng(rows)
    check(draw(rows, rows, 9001),
          temperature=rng.choice([0.0, 0.5, 1.0, 2.0], rows), top_k=rng.choice([0, 1, 5, 100, 5000], rows),
          top_p=rng.choice([1.0, 0.95, 0.5, 0.01], rows), min_p=rng.choice([0.0, 0.02, 0.5], rows),
          uniform=rng.random(rows).astype(np.float32))


@pytest.mark.parametrize("uniform", [0.0, 0.25, 1 - 2.0 ** -24])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=5), dict(top_p=0.3), dict(top_k=3000, top_p=0.5)])
def test_equal_logits_go_by_index(cuda, uniform, settings):
    """One value everywhere (also the lowest of the type, a common mask), and few distinct values."""
    for value in (0.0, -torch.finfo(torch.float32).max, 3.0):
        check(torch.full((2, 5000), value, device="cuda"), uniform=uniform, **settings)
    check(torch.randint(0, 3, (4, 40000), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).float(),
          uniform=uniform, **settings)


def test_zeros_of_both_signs_are_equal(cuda):
    x = torch.zeros(1, 64, device="cuda")
    x[0, :40] = -0.0
    check(x, top_k=2, uniform=0.75)
    check(x, temperature=0.0)


@pytest.mark.parametrize("mask", [-float("inf"), -torch.finfo(torch.float32).max, -1e9])
def test_masked_entries(cuda, mask):
    """A grammar's mask: all but a few entries out; k beyond what is left."""
    x = draw(8, 6, 3001)
    keep = torch.rand(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(2)) < 0.003
    keep[:, 5] = True
    x = torch.where(keep, x, mask)
    for settings in (dict(), dict(top_k=50), dict(top_p=0.99), dict(top_k=2000, top_p=0.9), dict(temperature=0.0)):
        for u in (0.0, 0.6, 1 - 2.0 ** -24):
            tokens = check(x, uniform=u, **settings)
            assert all(bool(keep[r, t]) for r, t in enumerate(tokens))


def test_row_with_nothing_left(cuda):
    x = draw(9, 3, 500)
    x[1] = -float("inf")
    for settings in (dict(), dict(top_k=4, top_p=0.5), dict(temperature=0.0)):
        tokens = check(x, **settings)
        assert tokens[1] == -1


def test_strided_and_unaligned_rows(cuda):
    for dtype in (torch.float32, torch.bfloat16):
        wide = draw(10, 7, 1100).to(dtype)
        for view in (wide[:, 3:1002], wide[::2, 1:], wide[1:2, 5:6], wide.flatten()[:1100 * 7 - 1].as_strided((3, 1001), (2001, 1), 1)):
            for settings in (dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.7)):
                check(view, uniform=0.77, **settings)


def test_distribution(cuda):
    """Evenly spaced uniforms give every token its share of the draws, but for one draw at each border."""
    n = 20000
    x = torch.tensor([0.3, -1.0, 2.0, 1.1, 0.0], device="cuda").expand(n, 5)
    u = (np.arange(n) + 0.5) / n
    tokens, chances, status, _ = run(x, uniform=u.astype(np.float32))
    w = np.exp(x[0].double().cpu().numpy())
    assert status == 0
    assert np.all(np.abs(np.bincount(tokens, minlength=5) - n * w / w.sum()) <= 2)


def test_bad_values_and_settings(cuda):
    x = draw(11, 6, 300)
    for value in (float("nan"), float("inf")):
        y = x.clone()
        y[2, 299] = value
        tokens, chances, status, _ = run(y)
        assert status == 2 and tokens[2] == -1 and chances[2] == 0 and (np.delete(tokens, 2) >= 0).all()
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
                dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(top_p=float("nan")), dict(min_p=1.01),
                dict(min_p=float("nan")), dict(uniform=1.0), dict(uniform=-0.1), dict(uniform=float("nan"))):
        key, value = next(iter(bad.items()))
        rows = np.array([dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniform=0.5)[key]] * 6)
        rows = rows.astype(np.float64) if key != "top_k" else rows
        rows[4] = value
        tokens, chances, status, _ = run(x, **{key: rows})
        assert status == 1 and tokens[4] == -1 and (np.delete(tokens, 4) >= 0).all(), bad


def test_refusals(cuda):
    x = draw(12, 2, 64)
    v = dict(temperature=torch.ones(2), top_k=torch.zeros(2, dtype=torch.int32), top_p=torch.ones(2),
             min_p=torch.zeros(2), uniform=torch.zeros(2))
    v = {k: t.cuda() for k, t in v.items()}
    ext = cuda_ops.extension()
    ext.sample_logits(x, **v)
    for logits, change in ((x.half(), {}), (x.t().contiguous().t(), {}), (x[0], {}), (x[:0], {}),
                           (torch.zeros(1, 262145, device="cuda").expand(2, -1), {}), (x.cpu(), {}),
                           (x, dict(top_k=v["top_k"].long())), (x, dict(uniform=v["uniform"].double())),
                           (x, dict(min_p=v["min_p"][:1])), (x, dict(top_p=v["top_p"].cpu()))):
        with pytest.raises(RuntimeError):
            ext.sample_logits(logits, **{**v, **change})
    x[1, 3] = float("nan")
    with pytest.raises(cuda_ops.ValidationError):
        cuda_ops.sample_logits(x, **v)
