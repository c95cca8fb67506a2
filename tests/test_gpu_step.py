"""Steps with drafted tokens as a program runs them: blocks and slots, rotations, append,
tree attention, sampling -- eagerly and captured in one graph -- against the definitions.

Tolerances: weights to BF16 2^-8, scores 2^-11, a BF16 output 2^-8; the rotations' own are covered by comparing against the rows that were appended.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops
from deepseekrpc_b200.rotary import rope_frequencies

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(192)
HEADS, IDX_HEADS, VOCAB, DRAFTS, BATCH = 16, 16, 5003, 5, 3
PARENTS = [-1, 0, 1, 0, 3]  # a chain 0-1-2 and the branch 3-4 of node 0
DEPTH = [0, 1, 2, 1, 2]


class Program:
    """A batch of requests and what a serving program keeps for it."""

    def __init__(self, seed):
        self.gen = torch.Generator("cuda").manual_seed(seed)
        blocks = 40
        self.kv = torch.full((blocks * 64, 576), float("nan"), device="cuda").bfloat16()
        self.index = torch.zeros((blocks * 64, 128), device="cuda").bfloat16()
        self.generations = torch.zeros(blocks * 64, dtype=torch.int64, device="cuda")
        self.table = torch.full((BATCH, 12), -1, dtype=torch.int32, device="cuda")
        self.held = torch.zeros(BATCH, dtype=torch.int32, device="cuda")
        self.ring = torch.randperm(blocks, generator=self.gen, device="cuda").to(torch.int32)
        self.state = torch.tensor([0, blocks, 0, 0], dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(BATCH, dtype=torch.int32, device="cuda")
        self.freq, self.mscale = rope_frequencies(64, scaling="yarn", factor=40.0)
        self.freq = self.freq.cuda()
        self.unembed = self.randn(HEADS * 512, VOCAB).bfloat16()
        self.sink = self.randn(HEADS)
        words = []
        for i, p in enumerate(PARENTS):
            words.append((words[p] if p >= 0 else 0) | 1 << i)
        self.masks = words
        self.mask = torch.tensor(words * BATCH, device="cuda")
        self.depth = torch.tensor(DEPTH * BATCH, dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.mirror = [np.zeros((0, 576)) for _ in range(BATCH)]  # each request's cached rows

    def randn(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda")

    def projections(self, tokens):
        return dict(q=self.randn(tokens, HEADS, 576).bfloat16(), idx_q=self.randn(tokens, IDX_HEADS, 128),
                    kv=self.randn(tokens, 576).bfloat16(), key=self.randn(tokens, 128).bfloat16(),
                    uniform=torch.rand(tokens, generator=self.gen, device="cuda"))

    def step(self, p, new, tokens, positions=None, drafts=False):
        """One pass over `tokens` new tokens; everything on the device."""
        ext = cuda_ops.extension()
        seq, position, slots, cu, visible, _ = ext.paged_plan(self.lengths, new, self.held, self.table, self.ring,
                                                              self.state, tokens, status=self.status)
        angle = position if positions is None else self.lengths[seq.long()] + positions
        x = [p["q"], p["idx_q"], p["kv"], p["key"]]
        ext.rope(x, x, angle, self.freq, [512, 64, 512, 64], [True, False, True, False], mscale=self.mscale,
                 status=self.status)
        expected = self.generations[slots.long()]
        appended = ext.append_kv_index(self.kv, self.index, self.generations, self.table, seq, position, expected,
                                       p["kv"], p["key"])
        out = dict(slots=slots, position=position, seq=seq, appended=appended)
        if drafts:
            out["attention"] = ext.tree_mla_decode(p["q"], self.kv, self.table, self.lengths, cu, self.mask, DRAFTS, SCALE,
                                                   sink=self.sink, status=self.status)[0]
            out["logits"] = out["attention"].reshape(tokens, -1).float() @ self.unembed.float() * 0.02
            rows = torch.ones(tokens, device="cuda")
            out["tokens"], out["chances"], _ = ext.sample_logits(out["logits"], rows * 0.8, (rows * 40).to(torch.int32),
                                                                 rows * 0.95, rows * 0.02, p["uniform"],
                                                                 status=self.status)
        return out

    def check(self, p, out):
        """A step with drafts against the 64-bit definitions."""
        assert int(self.status.item()) == 0 and int(out["appended"].item()) == 0
        lengths = self.lengths.tolist()
        for b in range(BATCH):
            at = slice(b * DRAFTS, (b + 1) * DRAFTS)
            rows = p["kv"][at].double().cpu().numpy()
            assert torch.equal(self.kv[out["slots"][at].long()], p["kv"][at])
            assert torch.equal(self.index[out["slots"][at].long()], p["key"][at])
            keys = np.concatenate([self.mirror[b][:lengths[b]], rows])
            q = p["q"][at].double().cpu().numpy()
            ref, _ = serving.tree_attention(q, keys, lengths[b], self.masks, self.sink.double().cpu().numpy(), SCALE)
            size = np.abs(keys).max()
            got = out["attention"][at].double().cpu().numpy()
            assert np.all(np.abs(got - ref) <= (2.0 ** -8 + 2.0 ** -11) * size + 2.0 ** -8 * np.abs(ref))
            assert np.linalg.norm(got - ref) <= 2.0 ** -7 * np.linalg.norm(ref)
        x = out["logits"].double().cpu().numpy()
        u = p["uniform"].cpu().numpy()
        for r in range(len(x)):
            token, chance = serving.sample(x[r], np.float32(0.8), 40, np.float32(0.95), np.float32(0.02), u[r])
            assert int(out["tokens"][r]) == token
            assert abs(float(out["chances"][r]) - chance) <= 2.0 ** -24 * chance + 2.0 ** -40

    def accept(self, p, accepted):
        """Keeps the first `accepted` nodes of each request's chain."""
        for b, m in enumerate(accepted):
            rows = p["kv"][b * DRAFTS:b * DRAFTS + m].double().cpu().numpy()
            self.mirror[b] = np.concatenate([self.mirror[b][:int(self.lengths[b])], rows])
        self.lengths += torch.tensor(accepted, dtype=torch.int32, device="cuda")


def prompts(program, lengths):
    new = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    p = program.projections(int(new.sum()))
    out = program.step(p, new, int(new.sum()))
    assert int(out["appended"].item()) == 0 and int(program.status.item()) == 0
    start = 0
    for b, n in enumerate(lengths):
        program.mirror[b] = p["kv"][start:start + n].double().cpu().numpy()
        start += n
    program.lengths += new


def test_steps_from_prompts_to_drafts(cuda):
    program = Program(1)
    prompts(program, [130, 63, 1])
    new = torch.full((BATCH,), DRAFTS, dtype=torch.int32, device="cuda")
    for accepted in ([3, 1, 2], [1, 1, 1], [2, 3, 1], [3, 3, 3]):
        p = program.projections(BATCH * DRAFTS)
        out = program.step(p, new, BATCH * DRAFTS, program.depth, drafts=True)
        program.check(p, out)
        program.accept(p, accepted)
    # finished requests give their blocks back
    none = torch.zeros(BATCH, dtype=torch.int32, device="cuda")
    cuda_ops.paged_plan(none, none, program.held, program.table, program.ring, program.state, 0)
    assert program.state[1].item() == 40 and torch.all(program.table == -1)
    assert sorted(program.ring.tolist()) == list(range(40))


def test_a_captured_step_replays(cuda):
    """The whole step in one graph; lengths, projections and numbers change between replays."""
    program, eager = Program(2), Program(2)
    for one in (program, eager):
        prompts(one, [100, 127, 30])
    new = torch.full((BATCH,), DRAFTS, dtype=torch.int32, device="cuda")
    p = program.projections(BATCH * DRAFTS)
    for key in p:  # the same stream of numbers for both
        eager.randn(*p[key].shape) if key != "uniform" else torch.rand(p[key].shape, generator=eager.gen, device="cuda")
    saved = [t.clone() for t in (program.held, program.table, program.ring, program.state, program.kv, program.index,
                                 program.generations)]
    program.step({k: v.clone() for k, v in p.items()}, new, BATCH * DRAFTS, program.depth, drafts=True)  # loads all kernels
    for t, s in zip((program.held, program.table, program.ring, program.state, program.kv, program.index,
                     program.generations), saved):
        t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = program.step(p, new, BATCH * DRAFTS, program.depth, drafts=True)
    for accepted in ([2, 3, 1], [3, 1, 2], [1, 2, 3]):
        fresh = eager.projections(BATCH * DRAFTS)
        for key in p:
            p[key].copy_(fresh[key])
        graph.replay()
        expect = eager.step(fresh, new, BATCH * DRAFTS, eager.depth, drafts=True)
        program.check(p, out)
        for key in ("slots", "position", "attention", "tokens", "chances"):
            assert torch.equal(out[key], expect[key]), key
        program.accept(p, accepted)
        eager.accept(fresh, accepted)
