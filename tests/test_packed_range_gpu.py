"""Attention over keys and values of 4 bits where its numbers are far apart: one key far above the
rest, values from tiny to large, steps of few bits; and what other requests left in the pages."""

import dataclasses

import pytest
import torch

from packed_refs import attention, quantize4
from test_packed_kv_gpu import by_entry, check_attention, rand, scene, whole_batch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
SCALE, Q0 = 0.125, 8.0          # a query of one element: a key's score is the key's first element


@pytest.fixture(scope="module")
def ops(gpu_device):
    from tokensprint_amd.kernels import load_hip_ops
    return load_hip_ops(gpu_device)


WALKS = {
    "whole items": dict(packed_whole=1 << 20, packed_few=1 << 30),
    "shares": dict(packed_whole=0, packed_few=1 << 30),
    "wavefronts": dict(packed_items=0, packed_few=1 << 30),
}


@pytest.fixture
def walk(ops):
    before = ops.dispatch
    yield lambda name: setattr(ops, "dispatch", dataclasses.replace(before, **WALKS[name]))
    ops.dispatch = before


def run(ops, q, k, v, batch, whole, table, cache, nkv):
    """(outputs, the float64 form's, both [T, nq, hd] in float64 on the host)"""
    ops.kv_store(k, v, whole, table, cache)
    sizes = dict(num_heads=q.shape[1], num_kv_heads=nkv, head_dim=q.shape[2], scale=SCALE, window=None)
    got = ops.paged_attention(q, batch, table, cache, **sizes)
    want, _ = attention(q, by_entry(quantize4(k), whole), by_entry(quantize4(v), whole), batch,
                        num_kv_heads=nkv, scale=SCALE)
    return got.double().cpu(), want


def relative(got, want):
    """The error's norm over the result's, the worst of all rows and heads."""
    return float(((got - want).norm(dim=-1) / want.norm(dim=-1).clamp(min=1e-30)).max())


# Norms of errors over norms of results.  bfloat16: the result's rounding, half a step (2^-8) at the most, and a
# float16 rounding of every weight (2^-11 each at the most, independent of each other; twice that is allowed).  float32: a score of up to 14 + 4, 26 in units of log2,
# is rounded twice (26 x 2 x 2^-24 x ln 2 = 2.2e-6 of a weight), the exponential once more, weights in two parts keep 22
# bits, and sums of up to 128 products are rounded to 2^-24 each, independently: below 1e-5 in all.
TOLERANCE = {BF16: 2.0 ** -8 + 2.0 ** -10, F32: 1e-5}


def peaked(device, dtype, *, nq, nkv, hd, spans, above, std, place, seed=0):
    batch, whole, table, cache = scene(device, nkv=nkv, hd=hd, page=16, spans=spans, seed=seed)
    k = torch.zeros(whole.num_tokens, nkv, hd, dtype=dtype, device=device)
    k[:, :, 0] = rand((whole.num_tokens, nkv), dtype, device, seed + 1)
    v = rand((whole.num_tokens, nkv, hd), dtype, device, seed + 2, std)
    first = 0
    for n in whole.q_lens:
        k[first + min(place, n - 1), :, 0] = above
        v[first + min(place, n - 1)] = 0
        first += n
    q = torch.zeros(batch.num_tokens, nq, hd, dtype=dtype, device=device)
    q[:, :, 0] = Q0
    return q, k, v, batch, whole, table, cache, nkv


@pytest.mark.parametrize("name", list(WALKS))
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("above,std,place", [(8, 0.02, 0), (12, 0.1, 0), (12, 0.02, 1777), (14, 0.02, 0), (14, 0.1, 3000),
                                             (10, 1e-3, 0), (14, 1e-3, 900), (12, 5e-3, 0)])
def test_one_key_of_no_value_far_above_the_rest(ops, gpu_device, walk, name, dtype, above, std, place):
    """The others' weights are small beside that key's, and are all that the result is made of."""
    walk(name)
    got, want = run(ops, *peaked(gpu_device, dtype, nq=4, nkv=2, hd=64, spans=[(4000, 1), (1800, 1)], above=above, std=std,
                                 place=place))
    worst = relative(got, want)
    assert worst <= TOLERANCE[dtype]


@pytest.mark.parametrize("name", list(WALKS))
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [128, 96])
def test_the_same_in_other_head_sizes(ops, gpu_device, walk, name, dtype, hd):
    walk(name)
    got, want = run(ops, *peaked(gpu_device, dtype, nq=6, nkv=2, hd=hd, spans=[(2500, 1), (700, 1)], above=12, std=5e-3,
                                 place=1))
    worst = relative(got, want)
    assert worst <= TOLERANCE[dtype]


@pytest.mark.parametrize("name", list(WALKS))
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rising", [True, False])
def test_values_that_grow_or_shrink_along_the_context(ops, gpu_device, walk, name, dtype, rising):
    """Steps from 2^-14 to the largest of float16, with most weight on the tokens of small values."""
    walk(name)
    args = list(peaked(gpu_device, dtype, nq=4, nkv=2, hd=64, spans=[(3000, 1)], above=1, std=1.0, place=0))
    n = args[4].num_tokens
    exponent = torch.linspace(-10, 18, n, device=gpu_device)
    if not rising:
        exponent = exponent.flip(0)
    args[2] = (args[2].float() * torch.exp2(exponent.round())[:, None, None]).clamp(-6e5, 6e5).to(dtype)
    # a score of -ln 2 for every doubling: all tokens bring about as much to the sum
    args[1] = args[1].clone()
    args[1][:, :, 0] = (args[1][:, :, 0].float() - exponent.round()[:, None] * 0.6931).to(dtype)
    got, want = run(ops, *args)
    # (scores from -13 - 4 to 7 + 4, 41 apart in units of log2: half as much again as above)
    worst = relative(got, want)
    assert worst <= (TOLERANCE[BF16] if dtype is BF16 else 1.5e-5)


def assert_pages_are_of_no_consequence(ops, gpu_device, args, dtype):
    cache, results = args[6], []
    everything = whole_batch(gpu_device, [cache.num_pages * 16],
                             torch.arange(cache.num_pages, dtype=torch.int32, device=gpu_device)[None])
    for size in (1e-3, 3e4):
        left = rand((everything.num_tokens, 2, 64), dtype, gpu_device, 9, size)
        ops.kv_store(left, left, everything, everything.tables[0], cache)
        results.append(run(ops, *args)[0])
    assert torch.equal(*results)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("name", list(WALKS))
def test_what_the_pages_held_before_is_of_no_consequence(ops, gpu_device, walk, name, dtype):
    """Tokens behind the last key in its block, and pages that are other requests', change no bit."""
    walk(name)
    args = peaked(gpu_device, dtype, nq=4, nkv=2, hd=64, spans=[(300, 1), (6, 1), (1505, 1)], above=14, std=1e-3, place=0)
    assert_pages_are_of_no_consequence(ops, gpu_device, args, dtype)


# ------------------------------------------------------------------ one wavefront an item, at the sizes it serves


@pytest.mark.parametrize("dtype,nq,nkv,hd,page", [
    (BF16, 8, 4, 128, 16), (BF16, 6, 2, 96, 16), (BF16, 6, 3, 80, 32), (BF16, 4, 2, 256, 16), (BF16, 20, 1, 128, 64),
    (F32, 8, 4, 128, 16), (F32, 4, 2, 96, 16), (F32, 4, 2, 256, 16)])
@pytest.mark.parametrize("options", [dict(), dict(window=70, keep_first=20), dict(softcap=9.0, sink=True)])
def test_a_wavefront_an_item(ops, gpu_device, walk, dtype, nq, nkv, hd, page, options):
    walk("wavefronts")
    options = dict(options)
    if options.get("sink"):
        options["sink"] = rand((nq,), F32, gpu_device, 31)
    check_attention(ops, gpu_device, nq=nq, nkv=nkv, hd=hd, page=page, dtype=dtype,
                    spans=[(400, 1), (0, 1), (30, 17), (0, 40), (255, 1)], **options)


@pytest.mark.parametrize("dtype,nkv,hd", [(BF16, 8, 128), (F32, 8, 128), (BF16, 12, 96)])
def test_more_items_than_a_workgroup_each(ops, gpu_device, dtype, nkv, hd):
    """More than 1,024 items by the dispatch's own rule, one of them long."""
    spans = [(900 if i == 57 else i % 45, 1) for i in range(131)]
    assert 131 * nkv > ops.dispatch.packed_items
    check_attention(ops, gpu_device, nq=nkv, nkv=nkv, hd=hd, page=16, spans=spans, dtype=dtype)


# ------------------------------------------------------------------ how near to exact


@pytest.mark.parametrize("name", list(WALKS))
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_ordinary_numbers_to_the_types_rounding(ops, gpu_device, walk, name, dtype, hd):
    """Norms: bfloat16 as TOLERANCE; float32: scores of up to some 6 as sums of hd products of numbers of 22 bits
    and more, rounded hd / 32 times a part (below 4 x 2^-24 x 6 x 1.44 in units of log2, 1.4e-6 of a weight), and the
    parts of TOLERANCE's that do not grow with scores."""
    walk(name)
    nq, nkv = 4, 2
    batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=[(800, 1), (1999, 1), (3, 1)])
    k, v = rand((whole.num_tokens, nkv, hd), dtype, gpu_device, 1), rand((whole.num_tokens, nkv, hd), dtype, gpu_device, 2)
    q = rand((batch.num_tokens, nq, hd), dtype, gpu_device, 3, 1.0 if hd == 64 else 0.7)
    got, want = run(ops, q, k, v, batch, whole, table, cache, nkv)
    worst = relative(got, want)
    assert worst <= (TOLERANCE[BF16] if dtype is BF16 else 4e-6)
