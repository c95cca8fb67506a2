"""Requests that continue one prompt, as a program runs them: the prompt kept in a row of its
own, forks, drafted steps in one graph (blocks and slots, rotations, append, attention over
the common prompt), a request cut back into what it shares, the prompt's row given up, the
pool compacted -- against the definitions.

Tolerances: weights to BF16 2^-8, scores 2^-11, a BF16 output 2^-8, as in test_gpu_step.py;
copied and appended rows are compared bit for bit.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops
from deepseekrpc_b200.rotary import rope_frequencies
from test_sharing_host import consistent

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(192)
HEADS, REQUESTS, DRAFTS, BLOCKS = 32, 6, 3, 64
KEPT = REQUESTS  # the table row that keeps the prompt
WORDS = [1, 3, 5]  # node 0, its children 1 and 2
DEPTH = [0, 1, 1]


class Program:
    def __init__(self, seed):
        self.gen = torch.Generator("cuda").manual_seed(seed)
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
        self.kv = torch.full((BLOCKS * 64, 576), float("nan"), device="cuda").bfloat16()
        self.index = torch.zeros((BLOCKS * 64, 128), device="cuda").bfloat16()
        self.generations = torch.zeros(BLOCKS * 64, dtype=torch.int64, device="cuda")
        self.held, self.lengths, self.shares = i32(REQUESTS + 1), i32(REQUESTS + 1), i32(BLOCKS)
        self.table = torch.full((REQUESTS + 1, 12), -1, dtype=torch.int32, device="cuda")
        self.ring = torch.randperm(BLOCKS, generator=self.gen, device="cuda").to(torch.int32)
        self.state = torch.tensor([0, BLOCKS, 0, 0], dtype=torch.int32, device="cuda")
        self.prefix, self.holder, self.status = i32(REQUESTS), i32(REQUESTS), i32(1)
        self.freq = rope_frequencies(64)[0].cuda()
        self.sink = torch.randn(HEADS, generator=self.gen, device="cuda")
        self.masks = torch.tensor(WORDS * REQUESTS, device="cuda")
        self.depth = torch.tensor(DEPTH * REQUESTS, dtype=torch.int32, device="cuda")
        self.mirror = [np.zeros((0, 576)) for _ in range(REQUESTS + 1)]  # each row's cached rows

    @property
    def tables(self):
        return self.held, self.table, self.ring, self.state, self.shares

    def projections(self, tokens):
        randn = lambda *shape: torch.randn(shape, generator=self.gen, device="cuda").bfloat16()  # noqa: E731
        return dict(q=randn(tokens, HEADS, 576), kv=randn(tokens, 576), key=randn(tokens, 128))

    def append(self, p, new, tokens, rows, depth=None):
        """Blocks, rotations and rows for the new tokens of the first `rows` table rows."""
        ext = cuda_ops.extension()
        seq, position, slots, cu, _, _ = ext.paged_plan(self.lengths[:rows], new, self.held[:rows], self.table[:rows],
                                                        self.ring, self.state, tokens, status=self.status)
        angle = position if depth is None else self.lengths[seq.long()] + depth
        x = [p["q"], p["kv"], p["key"]]
        ext.rope(x, x, angle, self.freq, [512, 512, 64], [True, True, False], status=self.status)
        appended = ext.append_kv_index(self.kv, self.index, self.generations, self.table[:rows], seq, position,
                                       self.generations[slots.long()], p["kv"], p["key"])
        return slots, cu, appended

    def step(self, p, new):
        slots, cu, appended = self.append(p, new, REQUESTS * DRAFTS, REQUESTS, self.depth)
        out = cuda_ops.extension().prefix_mla_decode(p["q"], self.kv, self.table, self.lengths[:REQUESTS], cu, self.masks,
                                                     DRAFTS, self.prefix, self.holder, SCALE, sink=self.sink,
                                                     status=self.status)[0]
        return dict(slots=slots, appended=appended, out=out)

    def prompt(self, lengths):
        new = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        p = self.projections(sum(lengths))
        _, _, appended = self.append(p, new, sum(lengths), REQUESTS + 1)
        assert int(appended) == int(self.status) == 0
        at = 0
        for b, n in enumerate(lengths):
            self.mirror[b] = np.concatenate([self.mirror[b], p["kv"][at:at + n].double().cpu().numpy()])
            at += n
        self.lengths += new

    def cut(self, lengths):
        self.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        moves, count = cuda_ops.paged_release(self.lengths, *self.tables)
        cuda_ops.paged_copy([self.kv, self.index], [self.generations], moves, count)
        self.mirror = [m[:n] for m, n in zip(self.mirror, lengths)]
        self.verify_rows()
        return int(count)

    def verify_rows(self):
        consistent(*(t.cpu().numpy() for t in self.tables))
        table = self.table.cpu().numpy()
        for b, rows in enumerate(self.mirror):
            at = [table[b, p // 64] * 64 + p % 64 for p in range(len(rows))]
            assert np.array_equal(self.kv[at].double().cpu().numpy(), rows), b

    def check(self, p, out):
        assert int(self.status) == int(out["appended"]) == 0
        sink = self.sink.double().cpu().numpy()
        for b in range(REQUESTS):
            at = slice(b * DRAFTS, (b + 1) * DRAFTS)
            keys = np.concatenate([self.mirror[b], p["kv"][at].double().cpu().numpy()])
            q = p["q"][at].double().cpu().numpy()
            ref, _ = serving.tree_attention(q, keys, len(self.mirror[b]), WORDS, sink, SCALE)
            got = out["out"][at].double().cpu().numpy()
            assert np.all(np.abs(got - ref) <= (2.0 ** -8 + 2.0 ** -11) * np.abs(keys).max() + 2.0 ** -8 * np.abs(ref))
            assert np.linalg.norm(got - ref) <= 2.0 ** -7 * np.linalg.norm(ref)

    def accept(self, p, accepted):
        """Keeps node 0, and node 1 behind it where two are accepted."""
        for b, m in enumerate(accepted):
            rows = p["kv"][b * DRAFTS:b * DRAFTS + m].double().cpu().numpy()
            self.mirror[b] = np.concatenate([self.mirror[b], rows])
        self.lengths[:REQUESTS] += torch.tensor(accepted, dtype=torch.int32, device="cuda")

    def share(self, prefix, holder):
        self.prefix.copy_(torch.tensor(prefix, dtype=torch.int32))
        self.holder.copy_(torch.tensor(holder, dtype=torch.int32))


def test_a_prompt_and_its_continuations(cuda):
    g = Program(1)
    g.prompt([0] * 5 + [70, 300])  # one request with a prompt of its own, and the kept one
    parent = torch.tensor([KEPT] * 5 + [-1, -1], dtype=torch.int32, device="cuda")
    g.lengths[:5] = torch.tensor([300, 300, 300, 300, 192], dtype=torch.int32, device="cuda")
    moves, count = cuda_ops.paged_fork(parent, g.lengths, *g.tables)
    assert int(count) == 4  # 192 tokens are whole blocks
    before = g.generations.clone()
    cuda_ops.paged_copy([g.kv, g.index], [g.generations], moves, count)
    assert int((g.generations - before).sum()) == 4 * (300 % 64)
    for b in range(5):
        g.mirror[b] = g.mirror[KEPT][:int(g.lengths[b])]
    g.verify_rows()

    new = torch.full((REQUESTS,), DRAFTS, dtype=torch.int32, device="cuda")
    g.share([300] * 4 + [192, 0], [KEPT] * 5 + [-1])
    p = g.projections(REQUESTS * DRAFTS)
    # loads the kernels; a first step, all of whose drafts are rejected
    first = g.step({k: v.clone() for k, v in p.items()}, new)
    assert int(g.status) == int(first["appended"]) == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = g.step(p, new)

    def replay(accepted):
        for k, v in g.projections(REQUESTS * DRAFTS).items():
            p[k].copy_(v)
        graph.replay()
        g.check(p, out)
        g.accept(p, accepted)

    replay([1, 2, 1, 2, 1, 1])
    replay([2, 1, 1, 2, 2, 1])
    # request 1 goes back to a place within what it shares, request 3 to one within its own
    lengths = g.lengths.tolist()
    lengths[1], lengths[3] = 150, 300
    assert g.cut(lengths) == 1
    g.share([300, 150, 300, 300, 192, 0], [KEPT] * 5 + [-1])
    replay([1, 2, 2, 1, 1, 2])
    # the prompt's row is given up: its blocks live on in the requests', one of which is read now
    lengths = g.lengths.tolist()
    lengths[KEPT] = 0
    assert g.cut(lengths) == 0
    g.share([300, 150, 300, 300, 192, 0], [2] * 5 + [-1])
    replay([2, 2, 1, 1, 2, 1])
    # two requests end, the others move together
    lengths = g.lengths.tolist()
    lengths[0] = lengths[5] = 0
    g.cut(lengths)
    moves, count = cuda_ops.paged_compact(*g.tables)
    cuda_ops.paged_copy([g.kv, g.index], [g.generations], moves, count)
    g.verify_rows()
    used = BLOCKS - int(g.state[1])
    assert int(g.table.max()) == used - 1 and int(count) > 0
    g.share([0, 150, 300, 300, 192, 0], [-1] + [2] * 4 + [-1])
    replay([1, 1, 2, 2, 1, 1])
    replay([1, 2, 1, 2, 1, 2])
    assert g.cut([0] * (REQUESTS + 1)) == 0
    assert int(g.state[1]) == BLOCKS and int(g.shares.abs().sum()) == 0
