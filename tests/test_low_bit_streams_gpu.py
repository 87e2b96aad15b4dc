"""Attention over keys and values of 4 bits and split products in 8 bits on several streams."""

import pytest
import torch

from test_packed_kv_gpu import heads_of, rand, scene
from tokensprint_amd.kernels.hip_ops import HipOps, KernelError

pytestmark = pytest.mark.gpu


def long_step(device, seed):
    """Arguments of a call whose keys are shared out over workgroups, and its queries."""
    batch, whole, table, cache = scene(device, nkv=2, hd=64, page=16, spans=[(4200 + 300 * seed, 1), (7, 1)], seed=seed)
    k, v = heads_of(whole, 2, 64, torch.bfloat16, device, 6 + seed)
    return (whole, k, v), rand((2, 4, 64), torch.bfloat16, device, 7 + seed), batch, table, cache


SIZES = dict(num_heads=4, num_kv_heads=2, head_dim=64, scale=0.125, window=None)


def test_a_refused_call_leaves_other_streams_counts_alone(gpu_device):
    """Another stream's workgroups may be counting themselves in while a call of this one is refused."""
    ops = HipOps(gpu_device)
    (whole, k, v), q, batch, table, cache = long_step(gpu_device, 0)
    ops.kv_store(k, v, whole, table, cache)
    torch.cuda.synchronize()
    other = torch.cuda.Stream(gpu_device)
    with torch.cuda.stream(other):
        want = ops.paged_attention(q, batch, table, cache, **SIZES)
    mine = ops.paged_attention(q, batch, table, cache, **SIZES)
    torch.cuda.synchronize()
    assert torch.equal(mine, want)
    theirs, own = ops._count_arrays[other.cuda_stream, 0], ops._count_arrays[0, 0]
    assert not theirs.any() and not own.any()                  # left as zeros by every launch
    theirs.fill_(3)
    own.fill_(3)
    off = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device=gpu_device)[1:].view(2, 4, 64)
    with pytest.raises(KernelError, match="aligned"):
        ops.paged_attention(off, batch, table, cache, **SIZES)
    torch.cuda.synchronize()
    assert bool((theirs == 3).all()) and not own.any()
    with torch.cuda.stream(other):
        ops.reset_scratch()
    torch.cuda.synchronize()
    assert not theirs.any()


def test_steps_on_streams_beside_each_other(gpu_device):
    """Two streams' steps in flight together, a reset and a refused call on a third in between."""
    ops = HipOps(gpu_device)
    made = []
    for i in range(2):
        (whole, k, v), q, batch, table, cache = long_step(gpu_device, i)
        ops.kv_store(k, v, whole, table, cache)
        made.append((q, batch, table, cache, ops.paged_attention(q, batch, table, cache, **SIZES), torch.cuda.Stream(gpu_device)))
    weight = ops.quantize_weight(rand((4096, 8192), torch.float32, gpu_device, 1))
    rows = ops.quantize_rows(rand((40, 8192), torch.float32, gpu_device, 2))
    product = ops.linear(rows, weight, torch.float32)
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for q, batch, table, cache, want, stream in made:
            with torch.cuda.stream(stream):
                got.append((ops.paged_attention(q, batch, table, cache, **SIZES), want))
                got.append((ops.linear(rows, weight, torch.float32), product))
        ops.reset_scratch()
        with pytest.raises(ValueError):
            ops.paged_attention(made[0][0], made[0][1], made[0][2], made[0][3], **dict(SIZES, scale=-1.0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)
