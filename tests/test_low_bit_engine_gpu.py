"""Engines with keys and values in 4 bits and weights in 8, operators together as a model uses them,
against the CPU engine whose plain operators quantise the same way."""

import pytest
import torch

import drives
from helpers import FUBE, LAYER_E, PALE, PINE, SISE, TINY, ZOLO, ZONO, random_prompt
from kernel_refs import TorchOps
from packed_refs import quantize4
from tokensprint_amd.engine import ModelRunner
from tokensprint_amd.engine.assemble import load_model, random_model
from tokensprint_amd.kernels.int8 import Int8Rows, Int8Weight, row_bytes
from tokensprint_amd.weights import write_random_model

pytestmark = pytest.mark.gpu


class LowBitOps(TorchOps):
    """The plain operators, with keys and values rounded to what 4 bits hold as they are stored and
    products of 8-bit numbers."""

    kv_bits = None

    def kv_store(self, k, v, batch, table, cache):
        if self.kv_bits:
            k, v = quantize4(k).float(), quantize4(v).float()
        super().kv_store(k, v, batch, table, cache)

    @staticmethod
    def _quantized(x, kind):
        scale = x.float().abs().amax(1) / 127
        codes = (x.double() / scale.double().clamp(min=1e-300)[:, None]).round()
        out = torch.zeros(x.shape[0], row_bytes(x.shape[1]), dtype=torch.int8)
        out[:, :x.shape[1]] = codes.to(torch.int8)
        return kind(out, scale, x.shape[1])

    def quantize_weight(self, weight):
        return self._quantized(weight, Int8Weight)

    def linear(self, x, weight, out_dtype):
        if not isinstance(weight, Int8Weight):
            return super().linear(x, weight, out_dtype)
        return (self._quantized(x, Int8Rows).values() @ weight.values().T).to(out_dtype)

    def norm_linear(self, resid, delta, norm_weight, eps, weight, out_dtype, silu_mul=False):
        if not isinstance(weight, Int8Weight):
            return super().norm_linear(resid, delta, norm_weight, eps, weight, out_dtype, silu_mul)
        resid = resid if delta is None else resid + delta.float()
        h = self.rmsnorm(resid, norm_weight, eps, torch.float32)
        return (self.linear_silu_mul if silu_mul else self.linear)(h, weight, out_dtype), resid


MODELS = {"qwen3": TINY["B"], "qwen3 windowed": TINY["C"], "palelix": PALE["B"], "zolorax": ZOLO["B"],
          "zonopel": ZONO["B"], "pinedra": PINE["B"], "fubepel": FUBE["B"], "sisepel": SISE["B"]}


@pytest.fixture(scope="module", params=list(MODELS))
def folder(request, tmp_path_factory):
    cfg, seed, _ = MODELS[request.param]
    d = tmp_path_factory.mktemp("low_bit")
    write_random_model(d, cfg, seed, torch.float32)
    vocab = cfg.get("vocab_size") or cfg["vocab"]
    return d, {f"r{i}": random_prompt(n, vocab, 100 + i) for i, n in enumerate([5, 40, 1, 64, 23])}


@pytest.mark.parametrize("kv_bits,weight_bits", [(4, None), (None, 8), (4, 8)])
def test_models(gpu_device, folder, kv_bits, weight_bits):
    d, requests = folder

    def run(device, ops, kv=None, weights=None):
        _, model = load_model(d, "float32", device, ops=ops, weight_bits=weights)
        runner = ModelRunner(model, page_size=16, num_pages=16, num_slots=4, kv_bits=kv)
        collected = drives.drive_mixed(runner, requests)
        return {rid: collected.stacked(rid)[0].float() for rid in requests}

    plain_ops = LowBitOps()
    plain_ops.kv_bits = kv_bits
    got = run(gpu_device, None, kv_bits, weight_bits)
    want = run("cpu", plain_ops, None, weight_bits)
    wide = run("cpu", TorchOps())
    for rid in requests:
        error, effect = (got[rid] - want[rid]).norm(), (want[rid] - wide[rid]).norm()
        # Both sides round the same numbers to the same few bits, but for those that float32's roundings
        # put on the other side of a border.  One number of a row of K that goes the other way moves the
        # row's product by a scale times a column, where the roundings of all (uniform, a twelfth of a
        # scale squared each) move it by sqrt(K / 12) of those: sqrt(12 / 96) = 0.35 of what 8 bits
        # change, here, for a token and those that see it (0.35 met in one request of 35, 1e-5 in most).
        # Two such numbers in a token: 0.5.
        assert error <= 0.5 * effect + 1e-4 * want[rid].norm(), (rid, float(error), float(effect))


@pytest.mark.parametrize("graphs", [False, True])
def test_the_engine_generates(gpu_device, tmp_path, graphs):
    """Two layers of the 0.6B shape: captured decode steps draw the tokens of eager ones."""
    from tokensprint_amd.config import Config, SamplingParams
    from tokensprint_amd.engine.llm_engine import LLMEngine
    _, model = random_model(LAYER_E, 4, "bfloat16", gpu_device, weight_bits=8)
    prompts = [random_prompt(n, LAYER_E["vocab_size"], n) for n in (3, 40, 100, 17)]
    engine = LLMEngine(model, Config(model=str(tmp_path), max_model_len=160, kvcache_block_size=16, num_kvcache_blocks=64,
                                     max_num_seqs=4, max_num_batched_tokens=64, chunked_prefill=True, kv_bits=4,
                                     enforce_eager=not graphs, enable_prefix_caching=graphs))
    assert engine.runner.storage.views[0].k_pages.dtype == torch.uint8
    out = engine.generate(prompts, SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True), use_tqdm=False)
    assert [len(o) for o in out] == [20] * 4
    again = engine.generate(prompts, SamplingParams(temperature=0.0, max_tokens=20, ignore_eos=True), use_tqdm=False)
    if not graphs:
        assert again == out          # (cached prefixes cut portions elsewhere: sums in another order)
    assert all(0 <= t < LAYER_E["vocab_size"] for o in out + again for t in o)


def test_weight_bits_refused(gpu_device):
    with pytest.raises(ValueError, match="8 bits"):
        random_model(TINY["B"][0], 1, "bfloat16", gpu_device, weight_bits=4)


def test_what_a_model_with_8_bit_weights_reads(gpu_device):
    _, wide = random_model(LAYER_E, 4, "bfloat16", gpu_device)
    _, low = random_model(LAYER_E, 4, "bfloat16", gpu_device, weight_bits=8)
    table = LAYER_E["vocab_size"] * LAYER_E["hidden_size"] * 2
    assert 0.5 < (low.step_weight_bytes() - table) / (wide.step_weight_bytes() - table) < 0.51
