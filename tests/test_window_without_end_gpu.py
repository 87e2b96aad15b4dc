"""A window longer than any sequence is no window, whatever number says so."""

import pytest
import torch

from scenarios import paged_scenario
from test_packed_kv_gpu import heads_of, rand, scene

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_device):
    from tokensprint_amd.kernels import load_hip_ops
    return load_hip_ops(gpu_device)


@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 31, 1 << 32, 10 ** 10])
@pytest.mark.parametrize("spans", [[(70, 1), (5, 1)], [(70, 20), (0, 9)]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_windows_past_32_bits(ops, gpu_device, window, spans, dtype):
    sizes = dict(num_heads=4, num_kv_heads=2, head_dim=64, scale=0.125)
    batch, wide, table, _ = paged_scenario(gpu_device, dtype, nkv=2, hd=64, page_size=16, spans=spans)
    q = rand((batch.num_tokens, 4, 64), dtype, gpu_device, 3)
    assert torch.equal(ops.paged_attention(q, batch, table, wide, window=window, **sizes),
                       ops.paged_attention(q, batch, table, wide, window=None, **sizes))
    batch, whole, table, cache = scene(gpu_device, nkv=2, hd=64, page=16, spans=spans)
    k, v = heads_of(whole, 2, 64, dtype, gpu_device, 4)
    ops.kv_store(k, v, whole, table, cache)
    assert torch.equal(ops.paged_attention(q, batch, table, cache, window=window, **sizes),
                       ops.paged_attention(q, batch, table, cache, window=None, **sizes))
