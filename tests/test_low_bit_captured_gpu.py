"""Captured steps over keys and values of 4 bits and weights of 8: lengths that move between
replays, and engine steps against the same steps run eagerly."""

import dataclasses

import pytest
import torch

from helpers import LAYER_E, random_prompt
from packed_refs import attention, quantize4
from test_packed_kv_gpu import by_entry, heads_of, rand, scene, whole_batch
from tokensprint_amd.engine import ModelRunner, StepEntry
from tokensprint_amd.engine.assemble import random_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_device):
    from tokensprint_amd.kernels import load_hip_ops
    return load_hip_ops(gpu_device)


# What four requests have cached in one replay after another (None: an idle lane): from whole items to shares and
# back, parts of other workgroups each time, one request alone.
LENGTHS = [[30, 5, 200, 17], [4000, 3900, 20, 3], [1, 3999, 1, None], [None, None, 3500, None], [700, 701, 702, 703],
           [None] * 4, [4000, 4000, 4000, 4000], [2, 9, 3999, 64]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("workgroups", [0, 7])
def test_lengths_that_move_between_replays(ops, gpu_device, dtype, workgroups):
    nq, nkv, hd, longest = 4, 2, 64, 4000
    batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=[(longest - 1, 1)] * 4)
    k, v = heads_of(whole, nkv, hd, dtype, gpu_device, 3)
    ops.kv_store(k, v, whole, table, cache)
    held = by_entry(quantize4(k), whole), by_entry(quantize4(v), whole)
    before = ops.dispatch
    if workgroups:
        ops.dispatch = dataclasses.replace(before, packed_workgroups=workgroups)
    try:
        static = whole_batch(gpu_device, [longest] * 4, table.clone(), [longest - 1] * 4)
        q = rand((4, nq, hd), dtype, gpu_device, 5)

        def call(b):
            return ops.paged_attention(q, b, b.tables[0], cache, num_heads=nq, num_kv_heads=nkv, head_dim=hd,
                                       scale=hd ** -0.5, window=None)

        call(static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(static)
        for turn, lengths in enumerate(LENGTHS + LENGTHS[::-1]):
            q.copy_(rand((4, nq, hd), dtype, gpu_device, 50 + turn))
            positions = torch.tensor([0 if n is None else n - 1 for n in lengths], dtype=torch.int32)
            static.positions.copy_(positions)
            static.ctx_len.copy_(positions + 1)
            static.tables[0].copy_(table)
            for e, n in enumerate(lengths):
                if n is None:
                    static.tables[0][e] = -1
            out.fill_(7.0)
            graph.replay()
            eager = call(static)
            torch.cuda.synchronize()
            assert torch.equal(out, eager), (turn, lengths)
            live = [e for e, n in enumerate(lengths) if n is not None]
            idle = [e for e in range(4) if e not in live]
            assert not out[idle].any()
            if not live:
                continue
            part = whole_batch(gpu_device, [lengths[e] for e in live], table[live], [lengths[e] - 1 for e in live])
            want, size = attention(q[live], [held[0][e] for e in live], [held[1][e] for e in live], part,
                                   num_kv_heads=nkv, scale=hd ** -0.5)
            # weights and results in bfloat16's steps (2^-11 and 2^-8); float32: scores of up to 20 as sums of 64
            # products (2e-5 of a weight at the most)
            bound = 2e-5 * size + (2.0 ** -11 * size + 2.0 ** -8 * want.abs() if dtype is torch.bfloat16 else 0) + 1e-6
            worst = float(((out[live].double().cpu() - want).abs() / bound).max())
            assert worst <= 1, (turn, lengths, worst)
    finally:
        ops.dispatch = before


@pytest.mark.parametrize("kv_bits,weight_bits", [(4, None), (None, 8), (4, 8)])
def test_captured_steps_are_eager_ones(gpu_device, kv_bits, weight_bits):
    """Two layers of the 0.6B shape in bfloat16, the same tokens in both: logits of every decode step."""
    _, model = random_model(LAYER_E, 4, "bfloat16", gpu_device, weight_bits=weight_bits)
    prompts = {f"r{i}": random_prompt(n, LAYER_E["vocab_size"], n) for i, n in enumerate((3, 40, 100, 17, 64))}
    wide, rows = None, {}
    for graphs, bits in ((False, kv_bits), (True, kv_bits), (False, None)):
        runner = ModelRunner(model, page_size=16, num_pages=64, num_slots=8, graph_max_len=192 if graphs else None,
                             kv_bits=bits)
        live = {rid: runner.manager.admit(rid) for rid in prompts}
        for rid, rc in live.items():
            runner.manager.extend(rc, len(prompts[rid]))
            runner.step([StepEntry(rc, prompts[rid], 0, [len(prompts[rid]) - 1])])
        got = []
        for step in range(12):
            entries = []
            for i, (rid, rc) in enumerate(live.items()):
                at = len(prompts[rid]) + step
                runner.manager.extend(rc, at + 1)
                entries.append(StepEntry(rc, [(97 * step + 13 * i) % LAYER_E["vocab_size"]], at, [0]))
            got.append(runner.step(entries).float().cpu().clone())
        if graphs:
            assert runner.graphs                       # the steps were replays
        if bits == kv_bits:
            rows[graphs] = torch.stack(got)
        wide = torch.stack(got)
    error = float((rows[True] - rows[False]).norm() / rows[False].norm())
    # The same kernels for the same numbers, but for products in bfloat16, whose float32 sums may come in another order
    # (the head's; without weights of 8 bits the layers' too, rounded to bfloat16 here and there the other way).
    assert error <= (1e-4 if weight_bits else 2.0 ** -6), error
    if kv_bits:                                        # and it is not the wide cache's numbers that are compared
        assert float((rows[True] - wide).norm() / wide.norm()) > 1e-3
