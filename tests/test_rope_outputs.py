"""The checked rotation returns the outputs it was given, whatever they came in (no GPU: the
extension's call is replaced by one that records its arguments)."""
from __future__ import annotations

import types

import torch

from deepseekrpc_b200 import cuda_ops


def test_outputs_from_an_iterator_are_returned(monkeypatch):
    seen = []

    def rope(x, out, *args, **settings):
        seen.append((x, out))
        return torch.zeros(1, dtype=torch.int32)

    monkeypatch.setattr(cuda_ops, "extension", lambda: types.SimpleNamespace(rope=rope))
    x, given = [torch.zeros(2, 4), torch.zeros(2, 8)], [torch.ones(2, 4), torch.ones(2, 8)]
    args = (torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.float64))
    for make in (list, tuple, iter):
        out = cuda_ops.rope(make(x), *args, offsets=[0, 0], interleaved=[True, True], out=make(given))
        assert len(out) == 2 and all(a is b for a, b in zip(out, given))
        assert all(a is b for a, b in zip(seen[-1][0], x)) and all(a is b for a, b in zip(seen[-1][1], given))
