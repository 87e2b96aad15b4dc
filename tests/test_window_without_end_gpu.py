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


@pytest.mark.parametrize("window", [1 << 31, (1 << 32) + 5, 10 ** 10])
def test_windows_past_32_bits_where_the_projection_merges(ops, gpu_device, monkeypatch, window):
    """A decode step whose key splits the output projection merges as it loads its rows."""
    from tokensprint_amd.kernels.stream import NormHint, UnmergedRows
    nq, nkv, hd, hidden, dtype = 16, 8, 128, 1024, torch.bfloat16
    batch, cache, table, _ = paged_scenario(gpu_device, dtype, nkv=nkv, hd=hd, page_size=16, spans=[(5000, 1), (2047, 1)])
    T = batch.num_tokens
    monkeypatch.setattr(ops, "merged_rows", 16)
    qkv = rand((T, (nq + 2 * nkv) * hd), dtype, gpu_device, 2)
    w_o = rand((hidden, nq * hd), dtype, gpu_device, 3, 0.05)
    hint = NormHint(torch.ones(hidden, device=gpu_device), 1e-6, rand((2 * 96, hidden), dtype, gpu_device, 4, 0.05), True)

    def run(window):
        o = ops.attend(qkv, batch, table, cache, True, defer_merge=True, num_heads=nq, num_kv_heads=nkv, kv_in_row=nkv,
                       head_dim=hd, q_weight=None, k_weight=None, eps=1e-6, cos_sin=None, scale=hd ** -0.5, window=window)
        assert isinstance(o, UnmergedRows)
        resid = torch.zeros(T, hidden, device=gpu_device)
        prepared = ops.linear_into_stream(o.view(T, nq * hd), w_o, resid, hint)
        assert prepared is not None and not o.is_merged
        return resid

    assert torch.equal(run(window), run(None))
