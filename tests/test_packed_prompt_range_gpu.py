"""Prompts' attention over keys and values of 4 bits where its numbers are far apart."""

import dataclasses

import pytest
import torch

from test_packed_kv_gpu import rand, scene
from test_packed_range_gpu import (BF16, F32, TOLERANCE, assert_pages_are_of_no_consequence, peaked, relative, run)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_device):
    """All portions by the kernel that makes tiles in LDS."""
    from tokensprint_amd.kernels import load_hip_ops
    ops = load_hip_ops(gpu_device)
    before = ops.dispatch
    ops.dispatch = dataclasses.replace(before, packed_few=0, packed_portion=1)
    yield ops
    ops.dispatch = before


# (as for single tokens, beside a float16 rounding of every key's and value's number: values' of 2^-11 at the most,
# independent of the weights' and of each other)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("above,std,place", [(8, 0.02, 0), (12, 0.1, 0), (12, 0.02, 1777), (14, 0.02, 0), (14, 0.1, 3000),
                                             (10, 1e-3, 0), (14, 1e-3, 900), (12, 5e-3, 0),
                                             (16.875, 0.05, 0), (16.875, 5e-3, 1000), (14.0625, 0.02, 0)])
def test_one_key_of_no_value_far_above_the_rest(ops, gpu_device, hd, above, std, place):
    got, want = run(ops, *peaked(gpu_device, BF16, nq=4, nkv=2, hd=hd, spans=[(4000, 24), (1800, 17)], above=above, std=std,
                                 place=place))
    worst = relative(got, want)
    assert worst <= TOLERANCE[BF16]


@pytest.mark.parametrize("hd", [64, 128])
def test_more_items_than_units(ops, gpu_device, hd):
    """Where items fill the card one set of wavefronts has all of an item's keys, else two share them."""
    spans = [(1200 + 3 * i, 2) for i in range(130)]
    assert 2 * len(spans) > ops._units
    got, want = run(ops, *peaked(gpu_device, BF16, nq=4, nkv=2, hd=hd, spans=spans, above=14, std=0.05, place=7))
    # The key's number is rounded to 11 bits: of a score of 14 (a step of 0.93310546875, a number of
    # 15 / 16 of it, 0.87478638, which becomes 0.875) that is 13.9966 x 2.441e-4 = 3.417e-3, by which all the others'
    # weights shrink together.
    worst = relative(got, want)
    assert worst <= TOLERANCE[BF16] + 3.43e-3


def test_what_the_pages_held_before_is_of_no_consequence(ops, gpu_device):
    args = peaked(gpu_device, BF16, nq=4, nkv=2, hd=64, spans=[(300, 23), (40, 30), (1505, 3)], above=14, std=1e-3, place=0)
    assert_pages_are_of_no_consequence(ops, gpu_device, args, BF16)


@pytest.mark.parametrize("hd", [64, 128])
def test_ordinary_numbers_to_the_types_rounding(ops, gpu_device, hd):
    nq, nkv = 4, 2
    batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=[(800, 30), (0, 20)])
    k, v = rand((whole.num_tokens, nkv, hd), BF16, gpu_device, 1), rand((whole.num_tokens, nkv, hd), BF16, gpu_device, 2)
    q = rand((batch.num_tokens, nq, hd), BF16, gpu_device, 3, 1.0 if hd == 64 else 0.7)
    got, want = run(ops, q, k, v, batch, whole, table, cache, nkv)
    # (a key's 11 bits too: hd independent roundings of 2^-11 |k q|, scores to 2^-9 of their deviation of 1)
    worst = relative(got, want)
    assert worst <= TOLERANCE[BF16] + 2.0 ** -9


@pytest.mark.parametrize("hd", [64, 128])
def test_steps_keep_their_bits(ops, gpu_device, hd):
    """Steps of 2^-14 to 2^-13, held in 10 to 11 bits; codes of 0 and 15 alone, so that numbers are not small beside
    float16's smallest ones where the steps are."""
    nq, nkv = 4, 2
    batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=[(600, 40), (0, 33)])
    T = whole.num_tokens
    size = (15 * 2.0 ** -14 * (1 + torch.rand(T, nkv, 1, generator=torch.Generator().manual_seed(1)))).to(gpu_device)
    on = (rand((T, nkv, hd), F32, gpu_device, 2) > 0).float()
    sign = rand((T, nkv, 1), F32, gpu_device, 3).sign()
    v = (size * on * sign).to(BF16)
    k = torch.zeros(T, nkv, hd, dtype=BF16, device=gpu_device)
    k[:, :, 0] = (15 * 2.0 ** -13 * rand((T, nkv), F32, gpu_device, 4).clamp(-1, 1)).to(BF16)
    q = torch.zeros(batch.num_tokens, nq, hd, dtype=BF16, device=gpu_device)
    q[:, :, 0] = 4 * 4096.0
    got, want = run(ops, q, k, v, batch, whole, table, cache, nkv)
    # as TOLERANCE; numbers have 11 bits from 2^-14 on (a key's, of 15 steps / 16: scores of up to 3.8 to 2^-11
    # at the most, 2e-3 of a weight, independent)
    worst = relative(got, want)
    assert worst <= 2.0 ** -8 + 2.0 ** -9


def one_channel_keys(whole, nkv, hd, device, seed, scores=None):
    """Keys of one element, which is the score that a query of one element gives (in 11 bits)."""
    k = torch.zeros(whole.num_tokens, nkv, hd, dtype=BF16, device=device)
    k[:, :, 0] = (rand((whole.num_tokens, nkv), F32, device, seed) + (0 if scores is None else scores[:, None])).to(BF16)
    return k


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("std", [3e-6, 1e-5, 1e-4, 1.0, 30.0, 3e3, 1e5])
def test_values_of_any_size(ops, gpu_device, hd, std):
    """From steps of a few of float16's smallest numbers to its largest."""
    batch, whole, table, cache = scene(gpu_device, nkv=2, hd=hd, page=16, spans=[(700, 40), (0, 33)])
    k = one_channel_keys(whole, 2, hd, gpu_device, 1)
    v = (rand((whole.num_tokens, 2, hd), F32, gpu_device, 2) * std).to(BF16)
    q = torch.zeros(batch.num_tokens, 4, hd, dtype=BF16, device=gpu_device)
    q[:, :, 0] = 8.0
    got, want = run(ops, q, k, v, batch, whole, table, cache, 2)
    # (and scores of up to 4 to 2^-11 of themselves, independent of each other: 2^-9 at the most)
    worst = relative(got, want)
    assert worst <= TOLERANCE[BF16] + 2.0 ** -9


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("std", [1e-5, 1e-3, 1.0, 300.0, 3e4])
def test_keys_of_any_size(ops, gpu_device, hd, std):
    """With queries that bring the scores back to ordinary ones."""
    batch, whole, table, cache = scene(gpu_device, nkv=2, hd=hd, page=16, spans=[(700, 40), (0, 33)])
    k = (rand((whole.num_tokens, 2, hd), F32, gpu_device, 1) * std).to(BF16)
    v = rand((whole.num_tokens, 2, hd), BF16, gpu_device, 2)
    q = (rand((batch.num_tokens, 4, hd), F32, gpu_device, 3) * (8 / hd ** 0.5 / std)).to(BF16)
    got, want = run(ops, q, k, v, batch, whole, table, cache, 2)
    # (hd independent roundings of 2^-11 |k q|: scores, of a deviation of 1, to 2^-9 at the most)
    worst = relative(got, want)
    assert worst <= TOLERANCE[BF16] + 2.0 ** -9


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed", "one large block"])
@pytest.mark.parametrize("sets", [1, 2])
def test_values_of_many_sizes_in_one_context(ops, gpu_device, hd, order, sets):
    """Blocks of 16 tokens whose steps lie on either side of every border between scales; scores fall by ln 2 for every
    doubling, so that all tokens bring about as much to the sum."""
    spans = [(1500, 40), (0, 33)] if sets == 2 else [(1500, 2), (90, 30)] + [(33 + i, 1) for i in range(130)]
    batch, whole, table, cache = scene(gpu_device, nkv=2, hd=hd, page=16, spans=spans)
    n = whole.num_tokens
    exponent = torch.linspace(-12, 17, n, device=gpu_device).round()
    if order == "falling":
        exponent = exponent.flip(0)
    elif order == "mixed":
        exponent = exponent[torch.randperm(n, generator=torch.Generator().manual_seed(5)).to(gpu_device)]
    elif order == "one large block":
        exponent = torch.full_like(exponent, -9)
        exponent[48:64] = 16
    k = one_channel_keys(whole, 2, hd, gpu_device, 1, -0.6931 * exponent)
    v = (rand((n, 2, hd), F32, gpu_device, 2) * torch.exp2(exponent)[:, None, None]).clamp(-6e5, 6e5).to(BF16)
    q = torch.zeros(batch.num_tokens, 4, hd, dtype=BF16, device=gpu_device)
    q[:, :, 0] = 8.0
    got, want = run(ops, q, k, v, batch, whole, table, cache, 2)
    # (scores of up to 12 + 4 to 2^-11 of themselves, independent of each other: 2^-7 at the most for any one weight,
    # a third of that as the deviation of all of them, twice that is allowed)
    worst = relative(got, want)
    assert worst <= TOLERANCE[BF16] + 2.0 ** -7 * 2 / 3


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sets", [1, 2])
@pytest.mark.parametrize("size,place", [(40.0, 33), (40.0, 2500), (1500.0, 33)])
def test_a_large_value_that_counts_little(ops, gpu_device, hd, sets, size, place):
    """A key far above the rest, and one far below it with values a thousand times the others' and more: the others, which
    are what the result is made of, keep the bits of their weights."""
    spans = [(3000, 24), (2600, 17)] if sets == 2 else [(2600 + i, 1) for i in range(130)]
    args = list(peaked(gpu_device, BF16, nq=4, nkv=2, hd=hd, spans=spans, above=14.0625, std=0.05, place=0))
    first = 0
    for n in args[4].q_lens:
        args[1][first + place, :, 0] = -14.0
        args[2][first + place] = (rand((2, hd), F32, gpu_device, 12 + first) * size).to(BF16)
        first += n
    got, want = run(ops, *args)
    # (2,600 others of 0.05 and weights around e: some 5 in all; that key's 1,500 e^-14 is 0.0012)
    worst = relative(got, want)
    assert worst <= TOLERANCE[BF16]
