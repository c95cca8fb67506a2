"""Where the amplitude of scaled rotary frequencies goes when only a part of a head is rotated."""
from __future__ import annotations

import numpy as np

from oracle import serving
from deepseekrpc_b200.rotary import rope_frequencies


def test_amplitude_on_the_attention_scale_reaches_all_columns():
    """64 of 192 columns rotated: as the rotation's mscale the amplitude grows their part of the
    score alone; its square on the attention scale grows the whole score."""
    freq, m = rope_frequencies(64, scaling="yarn", factor=40.0)
    rng = np.random.default_rng(1)
    q, k = rng.standard_normal((5, 1, 192)), rng.standard_normal((5, 1, 192))
    at = np.array([0, 7, 1000, 65536, 131071])
    turn = lambda x, amplitude: serving.rope(x, at, freq.numpy(), 128, True, amplitude)  # noqa: E731
    whole, plain = (turn(q, 1.0) * turn(k, 1.0)).sum(-1), (q[..., :128] * k[..., :128]).sum(-1)
    scale = 1 / np.sqrt(192)
    assert np.allclose(scale * (turn(q, m) * turn(k, m)).sum(-1), scale * (plain + m * m * (whole - plain)), atol=1e-12)
    recipe = m * m * scale
    assert np.allclose(recipe * whole, scale * m * m * (plain + (whole - plain)), atol=1e-12)
    assert abs(m * m - 1.8739) < 1e-4  # what the rotated part alone would grow by
