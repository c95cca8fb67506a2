"""A captured step whose number of drafted tokens changes between replays, with none at all
among them: the rows behind the last one are padding through every operator.

Tolerances as in a step with full rows: weights to BF16 2^-8, scores 2^-11, a BF16 output 2^-8.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import serving
from deepseekrpc_b200 import cuda_ops
from test_gpu_step import BATCH, DEPTH, DRAFTS, SCALE, Program, prompts

pytestmark = pytest.mark.gpu
ROWS = BATCH * DRAFTS


class Ragged(Program):
    def __init__(self, seed):
        super().__init__(seed)
        self.new = torch.zeros(BATCH, dtype=torch.int32, device="cuda")
        self.depths = torch.tensor(DEPTH, dtype=torch.int32, device="cuda")
        self.words = torch.tensor(self.masks, device="cuda")

    def drafted(self, p):
        ext = cuda_ops.extension()
        seq, position, slots, cu, _, _ = ext.paged_plan(self.lengths, self.new, self.held, self.table, self.ring,
                                                        self.state, ROWS, status=self.status)
        start = self.lengths[seq.clamp(min=0).long()]
        node = torch.where(seq >= 0, position - start, 0).long()
        angle = torch.where(seq >= 0, start + self.depths[node], -1)
        x = [p["q"], p["idx_q"], p["kv"], p["key"]]
        ext.rope(x, x, angle, self.freq, [512, 64, 512, 64], [True, False, True, False], mscale=self.mscale,
                 status=self.status)
        appended = ext.append_kv_index(self.kv, self.index, self.generations, self.table, seq, position,
                                       self.generations[slots.long()], p["kv"], p["key"])
        attention = ext.tree_mla_decode(p["q"], self.kv, self.table, self.lengths, cu, self.words[node], DRAFTS, SCALE,
                                        sink=self.sink, status=self.status)[0]
        logits = attention.reshape(ROWS, -1).float() @ self.unembed.float() * 0.02
        rows = torch.ones(ROWS, device="cuda")
        tokens, chances, _ = ext.sample_logits(logits, rows * 0.8, (rows * 40).to(torch.int32), rows * 0.95,
                                               rows * 0.02, p["uniform"], status=self.status)
        return dict(slots=slots, seq=seq, position=position, appended=appended, attention=attention, logits=logits,
                    tokens=tokens, chances=chances)


def test_a_captured_step_replays_with_any_number_of_drafts(cuda):
    program = Ragged(3)
    prompts(program, [100, 127, 30])
    p = program.projections(ROWS)
    kept = (program.held, program.table, program.ring, program.state, program.kv, program.index, program.generations)
    saved = [t.clone() for t in kept]
    program.drafted({k: v.clone() for k, v in p.items()})  # loads all kernels
    for t, s in zip(kept, saved):
        t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = program.drafted(p)
    for counts, accepted in (([5, 5, 5], [3, 1, 2]), ([2, 0, 4], [2, 0, 1]), ([0, 0, 0], [0, 0, 0]),
                             ([1, 5, 0], [1, 2, 0]), ([0, 0, 3], [0, 0, 3]), ([5, 5, 5], [1, 1, 1])):
        total = sum(counts)
        program.new.copy_(torch.tensor(counts))
        raw = program.projections(ROWS)
        for key in p:
            p[key].copy_(raw[key])
            if key != "uniform":
                p[key][total:] = float("nan")  # padding rows may hold anything
        kv, index = program.kv.clone(), program.index.clone()
        graph.replay()
        assert int(program.status.item()) == 0 and int(out["appended"].item()) == 0
        assert torch.all(out["seq"][total:] == -1) and torch.all(out["attention"][total:] == 0)
        assert all(torch.isnan(p[k][total:]).all() for k in ("q", "idx_q", "kv", "key"))
        # nothing of the pools changes but the new rows
        rows = out["slots"][:total].long()
        kv[rows], index[rows] = p["kv"][:total], p["key"][:total]
        same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))  # noqa: E731
        assert same(program.kv, kv) and same(program.index, index)
        freq = program.freq.cpu().numpy()
        at = 0
        for b, n in enumerate(counts):
            s, length = slice(at, at + n), int(program.lengths[b])
            at += n
            if n == 0:
                continue
            # the drafted nodes turn by their depth: one value of a key's rotation, in BF16
            angle = length + np.array(DEPTH[:n])
            ref = serving.rope(raw["kv"][s].double().cpu().numpy()[:, None], angle, freq, 512, True, program.mscale)[:, 0]
            size = np.abs(raw["kv"][s].double().cpu().numpy()).max() * 2 * program.mscale
            got = p["kv"][s].double().cpu().numpy()
            assert np.all(np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * size)
            keys = np.concatenate([program.mirror[b][:length], got])
            ref, _ = serving.tree_attention(p["q"][s].double().cpu().numpy(), keys, length, program.masks[:n],
                                            program.sink.double().cpu().numpy(), SCALE)
            got = out["attention"][s].double().cpu().numpy()
            assert np.all(np.abs(got - ref) <= (2.0 ** -8 + 2.0 ** -11) * np.abs(keys).max() + 2.0 ** -8 * np.abs(ref))
            assert np.linalg.norm(got - ref) <= 2.0 ** -7 * np.linalg.norm(ref)
            program.mirror[b] = np.concatenate([program.mirror[b][:length],
                                                p["kv"][s][:accepted[b]].double().cpu().numpy()])
        x, u = out["logits"].double().cpu().numpy(), p["uniform"].cpu().numpy()
        for r in range(total):
            token, chance = serving.sample(x[r], np.float32(0.8), 40, np.float32(0.95), np.float32(0.02), u[r])
            assert int(out["tokens"][r]) == token
            assert abs(float(out["chances"][r]) - chance) <= 2.0 ** -24 * chance + 2.0 ** -40
        program.lengths += torch.tensor(accepted, dtype=torch.int32, device="cuda")
