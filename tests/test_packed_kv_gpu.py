"""Keys and values held in 4 bits: what goes into the cache comes back as the format's values,
and attention over it against a plain form in 64 bits."""

import dataclasses

import pytest
import torch

from packed_refs import attention, quantize4
from scenarios import paged_scenario

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(gpu_device):
    from tokensprint_amd.kernels import load_hip_ops
    return load_hip_ops(gpu_device)


@pytest.fixture
def dispatch(ops):
    before = ops.dispatch
    yield lambda **kw: setattr(ops, "dispatch", dataclasses.replace(before, **kw))
    ops.dispatch = before


def rand(shape, dtype, device, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)


def scene(device, *, nkv, hd, page, spans, seed=0):
    """(batch of the spans' new tokens, batch of all their tokens, table, empty packed cache)"""
    from tokensprint_amd.cache import packed_cache
    batch, wide, table, _ = paged_scenario(device, torch.bfloat16, nkv=nkv, hd=hd, page_size=page,
                                           spans=spans, seed=seed, fill=False)
    whole = whole_batch(device, [s + n for s, n in spans], table)
    return batch, whole, table, packed_cache(wide.num_pages, nkv, page, hd, device)


def whole_batch(device, lengths, table, starts=None):
    """A batch of every entry's tokens [start, length)."""
    from tokensprint_amd.engine.batch import StepBatch
    starts = starts or [0] * len(lengths)
    lens = [n - s for n, s in zip(lengths, starts)]

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=device)

    T, q_start = sum(lens), [0]
    for n in lens:
        q_start.append(q_start[-1] + n)
    return StepBatch(
        num_tokens=T, num_entries=len(lens), num_logit_rows=0, token_ids=ints([0] * T),
        positions=ints([p for s, n in zip(starts, lengths) for p in range(s, n)]),
        entry_of_token=ints([e for e, n in enumerate(lens) for _ in range(n)]),
        q_start=ints(q_start), ctx_len=ints(lengths), slot_ids=ints([0] * len(lens)),
        logit_rows=ints([0]), tables=[table], q_lens=lens, starts=starts, max_q_len=max(lens),
        max_ctx_len=max(lengths))


def heads_of(whole, nkv, hd, dtype, device, seed, loud=4.0):
    """Keys and values of the batch's tokens; every eleventh channel of a key is louder."""
    k = rand((whole.num_tokens, nkv, hd), torch.float32, device, seed)
    k = (k * (1 + loud * (torch.arange(hd, device=device) % 11 == 3))).to(dtype)
    return k, rand((whole.num_tokens, nkv, hd), dtype, device, seed + 1, 0.6)


def by_entry(x, whole):
    return [part.cpu() for part in x.split(whole.q_lens)]


# ------------------------------------------------------------------ into the cache and back


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nkv,hd,page", [(2, 16, 16), (3, 48, 16), (1, 64, 32), (2, 80, 16), (8, 128, 16),
                                         (2, 192, 64), (1, 256, 16), (2, 112, 256)])
def test_store_and_read_back(ops, gpu_device, dtype, nkv, hd, page):
    spans = [(0, 1), (0, 37), (0, 16), (0, 70)]
    _, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=page, spans=spans)
    k, v = heads_of(whole, nkv, hd, dtype, gpu_device, 3)
    ops.kv_store(k, v, whole, table, cache)
    got_k, got_v = ops.kv_values(whole, table, cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.float32)
    # (a step of 11 bits times a whole number below 16 is exact in float32)
    assert torch.equal(got_k.double(), quantize4(k))
    assert torch.equal(got_v.double(), quantize4(v))
    in_bf16 = ops.kv_values(whole, table, cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.bfloat16)
    assert torch.equal(in_bf16[0], got_k.bfloat16()) and torch.equal(in_bf16[1], got_v.bfloat16())


@pytest.mark.parametrize("cuts", [[1, 2, 3, 4, 5, 6, 7], [3, 17, 18, 21, 40], [5, 6, 30], [16, 32], []])
def test_portions_cut_anywhere_leave_the_same_cache(ops, gpu_device, cuts):
    """Four tokens share words of values: what is written beside the others' bits stays theirs."""
    nkv, hd, lengths = 2, 96, [45, 23, 50]
    _, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=[(0, n) for n in lengths])
    k, v = heads_of(whole, nkv, hd, torch.bfloat16, gpu_device, 5)
    cache.k_pages.fill_(0x5a)                     # other requests' bytes
    cache.v_pages.fill_(0xa5)
    at = [min(c, 45) for c in [0] + cuts] + [45]
    parts = [t.split(lengths) for t in (k, v)]
    for lo, hi in zip(at, at[1:]):
        ends = [min(hi, n) for n in lengths]
        live = [e for e, n in enumerate(ends) if n > lo]
        if hi == 45:
            ends = lengths
            live = [e for e, n in enumerate(lengths) if n > lo]
        if not live:
            continue
        rows = table[live].contiguous()
        part = whole_batch(gpu_device, [ends[e] for e in live], rows, [lo] * len(live))
        ops.kv_store(torch.cat([parts[0][e][lo:ends[e]] for e in live]),
                     torch.cat([parts[1][e][lo:ends[e]] for e in live]), part, rows, cache)
    got = ops.kv_values(whole, table, cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.float32)
    assert torch.equal(got[0].double(), quantize4(k))
    assert torch.equal(got[1].double(), quantize4(v))


def test_tokens_written_one_at_a_time_touch_nobody_else(ops, gpu_device):
    nkv, hd = 1, 128
    batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=[(20, 1), (7, 1)])
    cache.k_pages.random_(0, 255)
    cache.v_pages.random_(0, 255)
    before = ops.kv_values(whole, table, cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.float32)
    bytes_before = cache.k_pages.clone(), cache.v_pages.clone()
    k, v = heads_of(batch, nkv, hd, torch.bfloat16, gpu_device, 8)
    ops.kv_store(k, v, batch, table, cache)
    after = ops.kv_values(whole, table, cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.float32)
    new = torch.zeros(whole.num_tokens, dtype=torch.bool, device=gpu_device)
    new[[20, 28]] = True
    for a, b, x in zip(after, before, (k, v)):
        assert torch.equal(a[~new].nan_to_num(), b[~new].nan_to_num())
        assert torch.equal(a[new].double(), quantize4(x))
    pages = {int(table[0, 1]), int(table[1, 0])}                 # that hold the two tokens
    for a, b in zip((cache.k_pages, cache.v_pages), bytes_before):
        for p in range(cache.num_pages):
            assert p in pages or torch.equal(a[p], b[p])


def test_values_a_format_of_4_bits_does_not_hold(ops, gpu_device):
    """NaN as zero, infinities and steps beyond float16 cut off, tiny groups as zeros; a group of one
    sign counts zero in; an all-zero group."""
    inf, nan = float("inf"), float("nan")
    rows = torch.zeros(8, 1, 128)
    g = torch.Generator().manual_seed(1)
    rows[0, 0] = torch.randn(128, generator=g)
    rows[0, 0, 5], rows[0, 0, 77] = nan, nan
    rows[1, 0, 3], rows[1, 0, 4] = inf, -1.0
    rows[2, 0, :64] = -inf
    rows[3, 0] = torch.randn(128, generator=g) * 3e38
    rows[4, 0] = torch.randn(128, generator=g) * 1e-9
    rows[5, 0] = torch.rand(128, generator=g) + 5
    rows[6, 0] = -rows[5, 0]
    _, whole, table, cache = scene(gpu_device, nkv=1, hd=128, page=16, spans=[(0, 8)])
    x = rows.to(gpu_device)
    ops.kv_store(x, x, whole, table, cache)
    got = ops.kv_values(whole, table, cache, num_kv_heads=1, head_dim=128, out_dtype=torch.float32)
    for values in got:
        assert torch.isfinite(values).all()
        assert torch.equal(values.double(), quantize4(x))


def test_a_token_without_a_page(ops, gpu_device):
    batch, whole, table, cache = scene(gpu_device, nkv=2, hd=64, page=16, spans=[(0, 20), (0, 5)])
    k, v = heads_of(whole, 2, 64, torch.bfloat16, gpu_device, 2)
    table = table.clone()
    table[0, 1] = -1
    ops.kv_store(k, v, whole, table, cache)
    got_k, got_v = ops.kv_values(whole, table, cache, num_kv_heads=2, head_dim=64, out_dtype=torch.float32)
    want_k, want_v = quantize4(k), quantize4(v)
    want_k[16:20], want_v[16:20] = 0, 0
    assert torch.equal(got_k.double(), want_k) and torch.equal(got_v.double(), want_v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,hd,extra", [(4, 2, 32, 0), (6, 1, 64, 16), (16, 8, 128, 0), (4, 2, 256, 8)])
@pytest.mark.parametrize("norm,rotate", [(True, True), (False, True), (True, False)])
def test_prepared_heads_are_those_of_a_wider_cache(ops, gpu_device, dtype, nq, nkv, hd, extra, norm, rotate):
    """Norm and rotation as the kernel for a cache of the activation type does them: the same
    queries, and the keys and values that one holds, in 4 bits."""
    spans = [(5, 9), (0, 18), (31, 1)]
    batch, wide, table, _ = paged_scenario(gpu_device, dtype, nkv=nkv, hd=hd, page_size=16, spans=spans,
                                           fill=False)
    from tokensprint_amd.cache import packed_cache
    cache = packed_cache(wide.num_pages, nkv, 16, hd, gpu_device)
    T = batch.num_tokens
    qkv = rand((T, (nq + 2 * nkv) * hd + extra), dtype, gpu_device, 4)
    w_q, w_k = (1 + rand((hd,), torch.float32, gpu_device, 5 + i, 0.2) if norm else None for i in range(2))
    angle = torch.arange(64, device=gpu_device)[:, None] * torch.rand(hd // 2, device=gpu_device)
    args = dict(num_heads=nq, num_kv_heads=nkv, head_dim=hd, q_weight=w_q, k_weight=w_k, eps=1e-5,
                cos_sin=(angle.cos(), angle.sin()) if rotate else None, row_extra=extra)
    want_q = ops.qk_norm_rope_store(qkv, batch, table, wide, **args)
    got_q = ops.qk_norm_rope_store(qkv, batch, table, cache, **args)
    assert torch.equal(got_q, want_q)
    pos = batch.positions.long()
    page = table[batch.entry_of_token.long(), pos // 16].long()
    k, v = ops.kv_values(batch, table, cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.float32)
    assert torch.equal(k.double(), quantize4(wide.k_pages[page, :, pos % 16]))
    assert torch.equal(v.double(), quantize4(wide.v_pages[page, :, :, pos % 16]))


@pytest.mark.parametrize("nq,nkv,hd", [(3, 3, 48), (6, 2, 80), (8, 2, 96), (4, 2, 176)])
def test_prepared_heads_of_other_sizes(ops, gpu_device, nq, nkv, hd):
    """Sums of squares in another order than the other kernel's: queries to a rounding, keys to a
    step where the rounding of one went the other way."""
    spans = [(5, 9), (0, 18), (31, 1)]
    batch, wide, table, _ = paged_scenario(gpu_device, torch.float32, nkv=nkv, hd=hd, page_size=16,
                                           spans=spans, fill=False)
    from tokensprint_amd.cache import packed_cache
    cache = packed_cache(wide.num_pages, nkv, 16, hd, gpu_device)
    qkv = rand((batch.num_tokens, (nq + 2 * nkv) * hd), torch.float32, gpu_device, 4)
    w_q, w_k = (1 + rand((hd,), torch.float32, gpu_device, 5 + i, 0.2) for i in range(2))
    angle = torch.arange(64, device=gpu_device)[:, None] * torch.rand(hd // 2, device=gpu_device)
    args = dict(num_heads=nq, num_kv_heads=nkv, head_dim=hd, q_weight=w_q, k_weight=w_k, eps=1e-5,
                cos_sin=(angle.cos(), angle.sin()))
    want_q = ops.qk_norm_rope_store(qkv, batch, table, wide, **args)
    got_q = ops.qk_norm_rope_store(qkv, batch, table, cache, **args)
    # float32: squares of up to 176 elements in another order, at most 176 x 2^-24 of their sum
    # (half of that of its root), and a few roundings more, of values up to 6
    torch.testing.assert_close(got_q, want_q, rtol=1e-5, atol=1e-5)
    pos = batch.positions.long()
    page = table[batch.entry_of_token.long(), pos // 16].long()
    k, v = ops.kv_values(batch, table, cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.float32)
    stored = wide.k_pages[page, :, pos % 16]
    # half a step of the group's span (2.5 to 8 of such keys, / 15) and the float16 step's rounding
    assert float((k - stored).abs().max()) < 0.51 * float(stored.abs().max()) * 2 / 15
    assert float((k.double() != quantize4(stored)).double().mean()) < 0.05
    assert torch.equal(v.double(), quantize4(wide.v_pages[page, :, :, pos % 16]))


# ------------------------------------------------------------------ attention


def check_attention(ops, device, *, nq, nkv, hd, page, spans, dtype, seed=0, **options):
    batch, whole, table, cache = scene(device, nkv=nkv, hd=hd, page=page, spans=spans, seed=seed)
    k, v = heads_of(whole, nkv, hd, dtype, device, seed + 10)
    cache.v_pages.random_(0, 255)                # what earlier owners of the pages left, made finite below
    cache.k_pages.random_(0, 255)
    finite = rand((cache.num_pages * page, nkv, hd), dtype, device, 77, 3.0)
    everything = whole_batch(device, [cache.num_pages * page],
                             torch.arange(cache.num_pages, dtype=torch.int32, device=device)[None])
    ops.kv_store(finite, -finite, everything, everything.tables[0], cache)
    ops.kv_store(k, v, whole, table, cache)
    q = rand((batch.num_tokens, nq, hd), dtype, device, seed + 20)
    scale = hd ** -0.5
    window = options.pop("window", None)
    got = ops.paged_attention(q, batch, table, cache, num_heads=nq, num_kv_heads=nkv, head_dim=hd,
                              scale=scale, window=window, **options)
    want, size = attention(q, by_entry(quantize4(k), whole), by_entry(quantize4(v), whole), batch,
                           num_kv_heads=nkv, scale=scale, window=window, **options)
    assert got.dtype == dtype and torch.isfinite(got).all()
    error = (got.double().cpu() - want).abs()
    # A weight times a step is rounded once (bfloat16: 2^-8 of it), the result once more.  In float32
    # what counts is the scores' error: up to 6 sums of group products of up to 64 x 31 x |q| <= 6,000,
    # each rounded (2^-24), times a step of up to 1.5 and the scale: below 5e-5 / sqrt(hd) x 60;
    # measured against 1e-4 of the values' size.
    # Beside that, codes enter as 16 + c and what their zeros take off is a sum of its own: sums of up to
    # 31 steps, each rounded once for every 32 keys and, in float32, every one of three parts.
    step = float(v.abs().max()) * 2 / 15
    rounded = 2 * (3 if dtype == torch.float32 else 1) * -(-batch.max_ctx_len // 32) * 2.0 ** -24 * 31 * step
    bound = rounded + (2.0 ** -8 * (size + want.abs()) + 1e-4 * size if dtype == torch.bfloat16 else 1e-4 * size)
    worst = float((error / (bound + 1e-7)).max())
    assert worst <= 1, worst
    return got


LONG = {"one": [(0, 700)], "behind": [(333, 400), (0, 65), (1, 16)], "beside": [(600, 1), (40, 129), (3, 1), (0, 300), (900, 2)]}


@pytest.mark.parametrize("spans", list(LONG))
@pytest.mark.parametrize("nq,nkv,hd,page", [(8, 4, 128, 16), (4, 1, 64, 32), (6, 2, 128, 64), (20, 1, 64, 16), (3, 3, 128, 256),
                                            (4, 2, 96, 16)])
@pytest.mark.parametrize("window", [None, 100])
def test_portions_of_prompts(ops, gpu_device, dispatch, spans, nq, nkv, hd, page, window):
    dispatch(packed_few=0)
    check_attention(ops, gpu_device, nq=nq, nkv=nkv, hd=hd, page=page, spans=LONG[spans], dtype=torch.bfloat16,
                    window=window)


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1e4, 1e30])
@pytest.mark.parametrize("few", [0, 512])
def test_queries_of_any_magnitude(ops, gpu_device, dispatch, scale, few):
    """A row of queries is brought to float16's range: whatever it was, and rows of zeros."""
    dispatch(packed_few=few)
    nq, nkv, hd = 4, 2, 64
    batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=[(30, 40), (50, 1)])
    k, v = heads_of(whole, nkv, hd, torch.bfloat16, gpu_device, 3)
    ops.kv_store(k, v, whole, table, cache)
    q = rand((41, nq, hd), torch.float32, gpu_device, 4)
    q[7] = 0
    q[:, :, 5] *= 1e-3
    for dtype in DTYPES:
        x = (q * scale).to(dtype)
        got = ops.paged_attention(x, batch, table, cache, num_heads=nq, num_kv_heads=nkv, head_dim=hd,
                                  scale=float(0.125 / scale), window=None)
        want, size = attention(x, by_entry(quantize4(k), whole), by_entry(quantize4(v), whole), batch,
                               num_kv_heads=nkv, scale=float(0.125 / scale))
        # as in check_attention, float32's bound without the sums' share
        bound = (2.0 ** -8 * (size + want.abs()) if dtype == torch.bfloat16 else 0) + 1e-4 * size + 1e-5
        assert bool(((got.double().cpu() - want).abs() <= bound).all())


SPANS = {
    "one key": [(0, 1)],
    "decode": [(40, 1), (0, 1), (255, 1), (126, 1), (31, 1), (300, 1)],
    "mixed": [(40, 1), (3, 50), (0, 33), (128, 17), (0, 1), (60, 2)],
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spans", list(SPANS))
@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 2, 16, 16), (3, 1, 48, 16), (8, 2, 64, 32), (6, 3, 80, 16),
                                            (16, 8, 128, 16), (8, 1, 128, 256), (20, 1, 96, 16),
                                            (4, 4, 160, 16), (6, 2, 192, 16), (5, 1, 224, 64), (4, 2, 256, 16)])
def test_attention(ops, gpu_device, dtype, spans, nq, nkv, hd, page):
    check_attention(ops, gpu_device, nq=nq, nkv=nkv, hd=hd, page=page, spans=SPANS[spans], dtype=dtype)


OPTIONS = {
    "window 1": dict(window=1), "window 40": dict(window=40), "chunk": dict(chunk=48),
    "sink": dict(sink=True), "window, first keys": dict(window=33, keep_first=5),
    "window, chunk": dict(window=70, chunk=64), "softcap": dict(softcap=4.0),
    "slopes": dict(slopes=True), "query temperature": dict(q_temp=(0.4, 32)),
    "all": dict(window=90, keep_first=40, softcap=9.0, slopes=True, q_temp=(0.2, 50), sink=True),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spans", ["decode", "mixed"])
@pytest.mark.parametrize("options", list(OPTIONS))
@pytest.mark.parametrize("walk", ["shares", "one workgroup", "whole items", "wavefronts", "portions"])
def test_attention_options(ops, gpu_device, dispatch, dtype, spans, options, walk):
    dispatch(packed_portion=1 if walk == "portions" else 1 << 20, packed_items=0 if walk == "wavefronts" else 1 << 20, packed_whole=1 << 20 if walk == "whole items" else 0,
             packed_workgroups={"shares": 0, "one workgroup": 1}.get(walk, 7), packed_few=0 if walk == "portions" else 512)
    kw = dict(OPTIONS[options])
    nq, nkv, hd = 6, 2, 64
    if kw.get("sink"):
        kw["sink"] = rand((nq,), torch.float32, gpu_device, 31)
    if kw.get("slopes"):
        kw["slopes"] = torch.rand(nq, device=gpu_device) * 0.1
    check_attention(ops, gpu_device, nq=nq, nkv=nkv, hd=hd, page=16, spans=SPANS[spans], dtype=dtype, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_contexts_in_shares(ops, gpu_device, dispatch, dtype):
    """Shares of unlike requests: one of a single key beside thousands."""
    spans = [(0, 1), (2999, 1), (1000, 1), (130, 1)]
    got = check_attention(ops, gpu_device, nq=4, nkv=2, hd=64, page=16, spans=spans, dtype=dtype)
    for workgroups in (1, 3, 24, 100, 400):
        dispatch(packed_workgroups=workgroups, packed_whole=0)
        again = check_attention(ops, gpu_device, nq=4, nkv=2, hd=64, page=16, spans=spans, dtype=dtype)
        twice = check_attention(ops, gpu_device, nq=4, nkv=2, hd=64, page=16, spans=spans, dtype=dtype)
        assert torch.equal(again, twice)             # the order of arrival changes nothing
        torch.testing.assert_close(again.float(), got.float(), rtol=2e-2, atol=2e-2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("options", list(OPTIONS))
def test_options_in_shares(ops, gpu_device, dispatch, dtype, options):
    """Long enough that items are shared: their parts meet what masks and scores add to them."""
    dispatch(packed_whole=0)
    kw = dict(OPTIONS[options])
    if kw.get("sink"):
        kw["sink"] = rand((6,), torch.float32, gpu_device, 31)
    if kw.get("slopes"):
        kw["slopes"] = torch.rand(6, device=gpu_device) * 0.01
    check_attention(ops, gpu_device, nq=6, nkv=2, hd=64, page=16, spans=[(2600, 1), (3, 1), (900, 1)], dtype=dtype, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nkv,spans", [
    (8, [(37 * i * i % 1400, 1) for i in range(40)]),               # more items than units: the longest first
    (1, [(3000 if i == 70 else i, 1) for i in range(100)]),         # more tiles than lanes, one of them shared
    (8, [(2500 if i == 3 else 40, 1) for i in range(33)]),          # one outlier among items that take turns
    (2, [(2000, 30), (5, 1), (0, 40), (700, 3)]),                   # portions of prompts in shares
])
def test_unlike_requests(ops, gpu_device, dispatch, dtype, nkv, spans):
    whole = check_attention(ops, gpu_device, nq=2 * nkv, nkv=nkv, hd=64, page=16, spans=spans, dtype=dtype)
    dispatch(packed_whole=0, packed_whole_many=0)
    again = check_attention(ops, gpu_device, nq=2 * nkv, nkv=nkv, hd=64, page=16, spans=spans, dtype=dtype)
    torch.testing.assert_close(again.float(), whole.float(), rtol=2e-2, atol=2e-2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nkv,hd", [(9, 128), (17, 64), (5, 256)])
def test_a_long_step_is_many_short_ones(ops, gpu_device, dtype, nkv, hd):
    """Steps of many tokens go round the waves otherwise: the same bytes, and the same numbers back."""
    spans = [(3, 4001), (0, 1), (18, 3), (1, 2222), (6, 1900)]
    batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=32, spans=spans)
    k, v = heads_of(batch, nkv, hd, dtype, gpu_device, 5)
    other = type(cache)(**{**vars(cache), "k_pages": cache.k_pages.clone(), "v_pages": cache.v_pages.clone()})
    ops.kv_store(k, v, batch, table, cache)
    first = 0
    for e, (start, n) in enumerate(spans):
        for lo in range(0, n, 333):
            hi = min(lo + 333, n)
            row = table[e:e + 1].contiguous()
            ops.kv_store(k[first + lo:first + hi], v[first + lo:first + hi],
                         whole_batch(gpu_device, [start + hi], row, [start + lo]), row, other)
        first += n
    assert torch.equal(cache.k_pages, other.k_pages) and torch.equal(cache.v_pages, other.v_pages)
    got = ops.kv_values(batch, table, cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.float32)
    assert torch.equal(got[0].double().cpu(), quantize4(k).cpu()) and torch.equal(got[1].double().cpu(), quantize4(v).cpu())
    part = whole_batch(gpu_device, [spans[0][0] + 200], table[:1].contiguous(), [spans[0][0]])
    few = ops.kv_values(part, table[:1].contiguous(), cache, num_kv_heads=nkv, head_dim=hd, out_dtype=torch.float32)
    assert torch.equal(few[0], got[0][:200]) and torch.equal(few[1], got[1][:200])


def test_one_key_stands_out(ops, gpu_device):
    """Scores far apart: the weight of one key is 1 wherever it lies, in whatever order maxima come."""
    nq, nkv, hd = 2, 1, 128
    batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=[(700, 1)])
    for place in (0, 17, 333, 699, 700):
        k, v = heads_of(whole, nkv, hd, torch.bfloat16, gpu_device, 3)
        q = rand((1, nq, hd), torch.bfloat16, gpu_device, 4)
        k[place] = 40 * q[:, 0].sign()
        ops.kv_store(k, v, whole, table, cache)
        out = ops.paged_attention(q, batch, table, cache, num_heads=nq, num_kv_heads=nkv, head_dim=hd,
                                  scale=hd ** -0.5, window=None)
        want = quantize4(v)[place, 0]
        # one weight, times a step, rounded to bfloat16, and the result once more
        assert bool(((out[0, 0].double() - want).abs() <= 2 ** -7 * want.abs() + 1e-5).all())


def test_idle_lanes_of_a_captured_step(ops, gpu_device):
    """Position 0 without a page: nothing is written, and zeros come out."""
    batch, whole, table, cache = scene(gpu_device, nkv=2, hd=64, page=16, spans=[(40, 1), (0, 1)])
    k, v = heads_of(whole, 2, 64, torch.bfloat16, gpu_device, 6)
    ops.kv_store(k, v, whole, table, cache)
    table = table.clone()
    table[1] = -1
    before = cache.k_pages.clone(), cache.v_pages.clone()
    qkv = rand((2, (4 + 4) * 64), torch.bfloat16, gpu_device, 7)
    out = ops.attend(qkv[1:].contiguous(), whole_batch(gpu_device, [1], table[1:]), table[1:], cache, True,
                     num_heads=4, num_kv_heads=2, kv_in_row=2, head_dim=64, q_weight=None, k_weight=None,
                     eps=0.0, cos_sin=None, scale=0.125, window=None)
    assert torch.equal(out, torch.zeros_like(out))
    assert torch.equal(cache.k_pages, before[0]) and torch.equal(cache.v_pages, before[1])


def test_counts_made_in_inference_mode_are_reset_outside(gpu_device):
    from tokensprint_amd.kernels.hip_ops import HipOps
    ops = HipOps(gpu_device)
    batch, whole, table, cache = scene(gpu_device, nkv=2, hd=64, page=16, spans=[(4000, 1), (7, 1)])
    k, v = heads_of(whole, 2, 64, torch.bfloat16, gpu_device, 6)
    q = rand((2, 4, 64), torch.bfloat16, gpu_device, 7)

    def call():
        return ops.paged_attention(q, batch, table, cache, num_heads=4, num_kv_heads=2, head_dim=64, scale=0.125,
                                   window=None)

    with torch.inference_mode():
        ops.kv_store(k, v, whole, table, cache)
        first = call()
    ops.reset_scratch()
    second = call()
    with torch.inference_mode():
        ops.reset_scratch()
        assert torch.equal(call(), second) and torch.equal(first, second)


def test_graphs_replayed_beside_each_other(ops, gpu_device):
    """Two captured steps on two streams, each with shares to merge, and eager calls between."""
    nq, nkv, hd, made = 4, 2, 64, []
    for i, spans in enumerate(([(4900, 1), (5, 1)], [(300, 1), (3200, 1)])):
        batch, whole, table, cache = scene(gpu_device, nkv=nkv, hd=hd, page=16, spans=spans, seed=i)
        k, v = heads_of(whole, nkv, hd, torch.bfloat16, gpu_device, 3 + i)
        ops.kv_store(k, v, whole, table, cache)
        q = rand((2, nq, hd), torch.bfloat16, gpu_device, 9 + i)
        call = lambda b=batch, t=table, c=cache, x=q: ops.paged_attention(     # noqa: E731
            x, b, t, c, num_heads=nq, num_kv_heads=nkv, head_dim=hd, scale=hd ** -0.5, window=None)
        want = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        made.append((graph, out, want, call))
    streams = [torch.cuda.Stream(gpu_device) for _ in made]
    for _ in range(4):
        for _, out, _, _ in made:
            out.zero_()
        torch.cuda.synchronize()
        for stream, (graph, _, _, _) in zip(streams, made):
            with torch.cuda.stream(stream):
                for _ in range(20):
                    graph.replay()
        eager = [call() for _, _, _, call in made]
        torch.cuda.synchronize()
        for (_, out, want, _), again in zip(made, eager):
            assert torch.equal(out, want) and torch.equal(again, want)


# ------------------------------------------------------------------ refusals


def test_refusals(ops, gpu_device):
    from tokensprint_amd.cache import packed_cache
    batch, whole, table, cache = scene(gpu_device, nkv=2, hd=64, page=16, spans=[(0, 20)])
    k, v = heads_of(whole, 2, 64, torch.bfloat16, gpu_device, 1)
    q = rand((20, 4, 64), torch.bfloat16, gpu_device, 2)
    sizes = dict(num_heads=4, num_kv_heads=2, head_dim=64, scale=0.125, window=None)
    for page, hd in ((8, 64), (24, 64), (48, 64), (16, 24), (16, 8), (16, 272)):
        with pytest.raises(ValueError):
            packed_cache(4, 2, page, hd, gpu_device)
    with pytest.raises(ValueError):                       # a cache of other heads
        ops.kv_store(k[:, :1].contiguous(), v[:, :1].contiguous(), whole, table, cache)
    with pytest.raises(ValueError):
        ops.paged_attention(q, whole, table, packed_cache(4, 2, 16, 128, gpu_device), **sizes)
    with pytest.raises(ValueError):                       # no positive scale
        ops.paged_attention(q, whole, table, cache, **dict(sizes, scale=0.0))
    with pytest.raises(ValueError):                       # a table too narrow
        ops.kv_store(k, v, whole, table[:, :1].contiguous(), cache)
    with pytest.raises(TypeError):
        ops.kv_values(whole, table, cache, num_kv_heads=2, head_dim=64, out_dtype=torch.float16)
    with pytest.raises(TypeError):
        ops.kv_store(k.half(), v.half(), whole, table, cache)
    wide = paged_scenario(gpu_device, torch.bfloat16, nkv=2, hd=64, page_size=16, spans=[(0, 20)])
    with pytest.raises(TypeError):
        ops.kv_values(wide[0], wide[2], wide[1], num_kv_heads=2, head_dim=64, out_dtype=torch.float32)
    from tokensprint_amd.kernels.hip_ops import KernelError
    off = torch.zeros(20 * 2 * 64 + 1, dtype=torch.bfloat16, device=gpu_device)[1:].view(20, 2, 64)
    with pytest.raises(KernelError, match="aligned"):
        ops.kv_store(off, off, whole, table, cache)
    with pytest.raises(ValueError):                       # operands on the host
        ops.kv_store(k.cpu(), v.cpu(), whole, table, cache)
