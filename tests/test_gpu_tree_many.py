"""Attention of more requests than a warp has lanes, long enough that the length of their
segments is searched, and short or many enough that it is not.  Tolerances: those of
test_gpu_serving_edges."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_serving_edges import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,heads,longest,most", [
    (33, 16, 6000, 3),    # one group a request, some cut
    (33, 64, 2500, 4),    # several groups
    (130, 16, 3000, 3),
    (64, 128, 700, 2),
    (65, 16, 20000, 1),   # few of them, long
    (2048, 16, 300, 1), (2049, 16, 100, 1),
])
def test_many_requests(cuda, batch, heads, longest, most):
    rng = np.random.default_rng(batch + heads)
    lengths = rng.integers(0, longest, batch)
    if longest == 20000:
        lengths[rng.permutation(batch)[:58]] %= 100
    counts = rng.integers(0, most + 1, batch)
    counts[0] = most
    attend(lengths.tolist(), counts.tolist(), heads, batch, padding=3)
