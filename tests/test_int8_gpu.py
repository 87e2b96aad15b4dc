"""Rows and weights in 8 bits and their products, against plain forms in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(gpu_device):
    from tokensprint_amd.kernels import load_hip_ops
    return load_hip_ops(gpu_device)


def rand(shape, dtype, device, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)


def quantize8(x):
    """(whole numbers, scales) of rows, in float64: the scale is float32's quotient."""
    scale = x.float().abs().amax(1) / torch.full((), 127.0, device=x.device)
    by = scale.double().where(scale > 0, torch.ones_like(scale, dtype=torch.float64))
    return (x.double() / by[:, None]).round(), scale.double()


def to_rounding(got, want, out_dtype):
    """float32: a whole number of up to 2^31 to 24 bits, and two products (3 x 2^-24); bfloat16 once more."""
    assert got.dtype == out_dtype
    rel = 4 * 2.0 ** -24 + (2.0 ** -8 if out_dtype == torch.bfloat16 else 0)
    worst = float(((got.double() - want).abs() / (want.abs() * rel + 1e-30)).max())
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 8), (2, 255), (7, 256), (33, 1000), (4, 4097), (9, 8192), (3, 12288),
                                 (2, 25600), (2, 40000)])
def test_rows(ops, gpu_device, dtype, M, K):
    x = rand((M, K), dtype, gpu_device, K, 3.0)
    x[-1, K // 2:] = 0
    got = ops.quantize_rows(x)
    numbers, scale = quantize8(x)
    assert got.shape == (M, K) and got.codes.dtype == torch.int8
    assert torch.equal(got.scales.double(), scale)
    # (numbers of scales to the nearest: a quotient that lies on the border to 2^-24 may go either way)
    off = (got.codes[:, :K].double() - numbers).abs()
    assert float(off.max()) <= 1 and float((off > 0).double().mean()) <= 1e-4
    assert not got.codes[:, K:].any()                            # zeros behind the row
    assert float((got.values().double() - x.double()).abs().max()) <= 0.5001 * float(scale.max())


def test_rows_of_zeros_and_of_what_is_no_number(ops, gpu_device):
    x = rand((6, 300), torch.float32, gpu_device, 1)
    x[1] = 0
    x[2, 7] = math.nan
    x[3, 299] = math.inf
    x[4, 0] = 3e38
    x[5] = 1e-40
    got = ops.quantize_rows(x)
    assert not got.codes[1].any() and float(got.scales[1]) == 0
    assert math.isnan(float(got.scales[2])) and math.isinf(float(got.scales[3]))
    w = ops.quantize_weight(rand((20, 300), torch.float32, gpu_device, 2))
    y = ops.linear(got, w, torch.float32)
    assert torch.equal(y[1], torch.zeros_like(y[1]))
    assert not torch.isfinite(y[2]).any() and not torch.isfinite(y[3]).any()
    # the others are finite wherever a float32 holds the product (rows of 3e38 times weights above 1.13 are not)
    want = (got.codes.double() @ w.codes.double().T) * got.scales.double()[:, None] * w.scales.double()
    held = want.abs() < 3.4e38
    assert held[[0, 1, 5]].all() and held[4].any()
    assert torch.isfinite(y[[0, 1, 4, 5]][held[[0, 1, 4, 5]]]).all()


def test_an_aligned_row_is_one_that_is_not(ops, gpu_device):
    """The walk an element at a time, for rows that begin anywhere: the same numbers."""
    x = rand((5, 1024), torch.bfloat16, gpu_device, 3)
    room = torch.empty(5 * 1024 + 1, dtype=torch.bfloat16, device=gpu_device)
    off = room[1:].view(5, 1024)
    off.copy_(x)
    a, b = ops.quantize_rows(x), ops.quantize_rows(off)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("delta", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K", [(1, 64), (5, 1000), (17, 1024), (3, 4096), (2, 5120), (2, 12288), (4, 77)])
def test_normed_rows(ops, gpu_device, delta, M, K):
    resid = rand((M, K), torch.float32, gpu_device, K)
    before = resid.clone()
    d = None if delta is None else rand((M, K), delta, gpu_device, K + 1, 0.3)
    w = 1 + rand((K,), torch.float32, gpu_device, K + 2, 0.2)
    rows, out = ops.norm_quantize_rows(resid, d, w, 1e-5)
    assert torch.equal(resid, before)
    stream = resid if d is None else resid + d.float()
    assert torch.equal(out, stream) and (d is not None or out is resid)
    x = stream.double()
    h = x / (x.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    # half a scale, and float32's roundings: a sum of K squares (K 2^-25 of the root at the most, K / 1,024 of that
    # in the kernel's order) and five products
    scale = rows.scales.double()[:, None]
    assert float(((rows.values().double() - h).abs() / scale).max()) <= 0.5 + 127 * (5 + K / 64) * 2.0 ** -24
    torch.testing.assert_close(scale[:, 0], h.abs().amax(1) / 127, rtol=(6 + K / 64) * 2.0 ** -24, atol=0)


SIZES = [(1, 16, 64), (1, 4096, 4096), (5, 33, 100), (16, 1000, 512), (17, 129, 1030), (33, 40, 4096), (64, 515, 768),
         (65, 515, 768), (65, 40, 200), (100, 7, 1024), (130, 1000, 1300), (300, 2048, 512), (513, 384, 5120), (2, 3, 1)]


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(ops, gpu_device, out_dtype, M, N, K):
    x, w = rand((M, K), out_dtype, gpu_device, 7), rand((N, K), torch.bfloat16, gpu_device, 8, 0.05)
    weight, rows = ops.quantize_weight(w), ops.quantize_rows(x)
    assert weight.shape == (N, K) and weight.numel() == N * K
    want = rows.values().double() @ weight.values().double().T
    sums = rows.codes.double() @ weight.codes.double().T
    want = sums * rows.scales.double()[:, None] * weight.scales.double()
    got = ops.linear(x, weight, out_dtype)
    to_rounding(got, want, out_dtype)
    assert torch.equal(ops.linear(rows, weight, out_dtype), got)


@pytest.mark.parametrize("tile", list(range(10)))
@pytest.mark.parametrize("M,N,K", [(1, 16, 1024), (70, 200, 1100), (300, 390, 1024)])
def test_product_in_every_tile(ops, gpu_device, tile, M, N, K):
    rows = ops.quantize_rows(rand((M, K), torch.float32, gpu_device, 7))
    weight = ops.quantize_weight(rand((2 * N, K), torch.float32, gpu_device, 8, 0.05))
    want = ops._int8_product(rows, weight, torch.float32, tile=9)
    sums = rows.codes.double() @ weight.codes.double().T
    to_rounding(want, sums * rows.scales.double()[:, None] * weight.scales.double(), torch.float32)
    assert torch.equal(ops._int8_product(rows, weight, torch.float32, tile=tile), want)
    pair = ops._int8_product(rows, weight, torch.float32, pair=True, tile=tile)
    gate, up = (sums * rows.scales.double()[:, None] * weight.scales.double()).chunk(2, 1)
    check_unit(pair, gate, up, torch.float32)


def check_unit(got, gate, up, out_dtype, limit=None, act="silu"):
    if limit is not None:
        g, u = gate.clamp(max=limit), up.clamp(-limit, limit)
        want, size = g * torch.sigmoid(1.702 * g) * (u + 1), g.abs() * (u.abs() + 1)
    elif act == "gelu_tanh":
        want = torch.nn.functional.gelu(gate, approximate="tanh") * up
        size = gate.abs() * up.abs()
    else:
        want, size = torch.nn.functional.silu(gate) * up, gate.abs() * up.abs()
    # 4 roundings of gate and of up, some ten of the unit, an exponential of a float32 argument up to 20 x
    # its rounding; of the product's size (tanh and the sigmoid lose what cancels)
    rel = 60 * 2.0 ** -24
    bound = rel * (size + want.abs()) + (2.0 ** -8 * want.abs() if out_dtype == torch.bfloat16 else 0) + 1e-30
    worst = float(((got.double() - want).abs() / bound).max())
    assert worst <= 1, worst


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("unit", [{}, {"limit": 1.5}, {"act": "gelu_tanh"}])
@pytest.mark.parametrize("M,N,K", [(1, 24, 64), (16, 1000, 512), (40, 129, 4096), (66, 515, 768), (300, 1024, 1000)])
def test_gate_and_up(ops, gpu_device, out_dtype, unit, M, N, K):
    x, w = rand((M, K), out_dtype, gpu_device, 7), rand((2 * N, K), torch.bfloat16, gpu_device, 8, 2 / K ** 0.5)
    weight, rows = ops.quantize_weight(w), ops.quantize_rows(x)
    sums = (rows.codes.double() @ weight.codes.double().T) * rows.scales.double()[:, None] * weight.scales.double()
    gate, up = sums.chunk(2, 1)
    check_unit(ops.linear_silu_mul(x, weight, out_dtype, **unit), gate, up, out_dtype, **unit)


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 12, 70])
@pytest.mark.parametrize("silu_mul", [False, True])
def test_norm_and_product(ops, gpu_device, out_dtype, M, silu_mul):
    """The two operators together, as a sub-layer begins with them."""
    K, N = 1024, 400
    resid, delta = rand((M, K), torch.float32, gpu_device, 1), rand((M, K), out_dtype, gpu_device, 2)
    norm = 1 + rand((K,), torch.float32, gpu_device, 3, 0.1)
    weight = ops.quantize_weight(rand((2 * N, K), torch.bfloat16, gpu_device, 4, 0.05))
    for d in (None, delta):
        rows, stream = ops.norm_quantize_rows(resid, d, norm, 1e-6)
        out, after = ops.norm_linear(resid, d, norm, 1e-6, weight, out_dtype, silu_mul=silu_mul)
        assert torch.equal(after, stream)
        want = (ops.linear_silu_mul if silu_mul else ops.linear)(rows, weight, out_dtype)
        assert torch.equal(out, want)


def test_no_rows(ops, gpu_device):
    w = ops.quantize_weight(rand((20, 64), torch.bfloat16, gpu_device, 1))
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=gpu_device)
    assert ops.linear(x, w, torch.bfloat16).shape == (0, 20)


def test_captured_and_replayed(ops, gpu_device):
    w = ops.quantize_weight(rand((640, 512), torch.bfloat16, gpu_device, 1, 0.05))
    x = rand((9, 512), torch.bfloat16, gpu_device, 2)
    ops.linear(x, w, torch.bfloat16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear(x, w, torch.bfloat16)
    for seed in range(3, 7):
        x.copy_(rand((9, 512), torch.bfloat16, gpu_device, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.linear(x, w, torch.bfloat16))


def test_refusals(ops, gpu_device):
    from tokensprint_amd.kernels.int8 import Int8Rows, Int8Weight
    w = ops.quantize_weight(rand((20, 64), torch.bfloat16, gpu_device, 1))
    x = rand((3, 64), torch.bfloat16, gpu_device, 2)
    with pytest.raises(ValueError):
        ops.linear(x[:, :32].contiguous(), w, torch.bfloat16)
    with pytest.raises(ValueError):
        ops.linear(x[:, ::2], w, torch.bfloat16)
    with pytest.raises(TypeError):
        ops.linear(x.half(), w, torch.bfloat16)
    with pytest.raises(TypeError):
        ops.linear(x, w, torch.float16)
    with pytest.raises(ValueError):                      # an odd number of gate and up rows
        ops.linear_silu_mul(x, ops.quantize_weight(rand((21, 64), torch.bfloat16, gpu_device, 1)), torch.bfloat16)
    with pytest.raises(ValueError):                      # numbers that are not in rows of 256 bytes
        ops.linear(Int8Rows(torch.zeros(3, 64, dtype=torch.int8, device=gpu_device),
                            torch.zeros(3, device=gpu_device), 64), w, torch.bfloat16)
    with pytest.raises(ValueError):
        ops.linear(x, Int8Weight(w.codes, w.scales[:-1], 64), torch.bfloat16)
    with pytest.raises(ValueError):
        ops.quantize_rows(torch.empty(1, 131073, device=gpu_device))
    with pytest.raises(ValueError):
        ops.quantize_weight(x.cpu())
    with pytest.raises(ValueError):
        ops.norm_quantize_rows(x.float(), x[:2], torch.ones(64, device=gpu_device), 1e-6)


@pytest.mark.parametrize("k", [64, 4096, 5000])
@pytest.mark.parametrize("rows", [1, 1000])
@pytest.mark.parametrize("top", [1e-35, 3e-37, 2e-38])
def test_rows_of_tiny_elements(ops, rows, k, top):
    """Scales below what a reciprocal in float32 has room for: still the nearest whole numbers."""
    x = (torch.rand(rows, k, dtype=torch.float64) * 2 - 1) * top
    x[:, 0] = top
    x = x.float()
    got = ops.quantize_rows(x.cuda())
    scale = got.scales.cpu().double()
    # (a scale below 2^-126 has fewer bits: half a step of 2^-149)
    assert ((scale - x.double().abs().amax(1) / 127).abs() <= scale * 2.0**-24 + 2.0**-150).all()
    ratio = x.double() / scale[:, None]
    assert ((got.codes.cpu()[:, :k].double() - ratio.clamp(-127, 127)).abs() <= 0.5).all()


@pytest.mark.parametrize("k", [8, 264, 2816, 4096, 8192, 8200])
@pytest.mark.parametrize("rows", [1, 2, 4, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_call_is_the_two_calls_to_the_bit(ops, rows, k, dtype):
    torch.manual_seed(k + rows)
    weight = ops.quantize_weight(torch.randn(2 * 77, k, device="cuda"))
    x = torch.randn(rows, k, device="cuda").to(dtype)
    assert torch.equal(ops.linear(x, weight, dtype), ops.linear(ops.quantize_rows(x), weight, dtype))
    assert torch.equal(ops.linear_silu_mul(x, weight, dtype),
                       ops.linear_silu_mul(ops.quantize_rows(x), weight, dtype))
    stream, w = torch.randn(rows, k, device="cuda"), torch.rand(k, device="cuda")
    for delta in (x, None):
        for pair in (False, True):
            before = stream.clone()
            out, after = ops.norm_linear(stream, delta, w, 1e-6, weight, dtype, silu_mul=pair)
            normed, want = ops.norm_quantize_rows(stream, delta, w, 1e-6)
            assert torch.equal(out, (ops.linear_silu_mul if pair else ops.linear)(normed, weight, dtype))
            assert torch.equal(after, want) and torch.equal(stream, before)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_one_call_with_a_row_that_is_not_finite(ops, value):
    """The other rows know nothing of it."""
    weight = ops.quantize_weight(torch.randn(48, 512, device="cuda"))
    x = torch.randn(3, 512, device="cuda")
    want = ops.linear(x, weight, torch.float32)
    x[1, 300] = value
    got = ops.linear(x, weight, torch.float32)
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    assert not torch.isfinite(got[1]).any()


@pytest.mark.parametrize("pair", [False, True])
@pytest.mark.parametrize("rows,n,k", [(17, 4096, 4096), (64, 1000, 2048), (33, 2048, 8192), (128, 515, 12288),
                                      (70, 96, 131072), (64, 4096, 5000)])
def test_products_split_along_the_rows(ops, rows, n, k, pair):
    """In parts that meet in memory, twice in a row, the bits are those of a tile that walks all of K; and so in
    a graph's replays beside eager calls."""
    torch.manual_seed(rows)
    weight = ops.quantize_weight(torch.randn(n * (2 if pair else 1), k, device="cuda"))
    x = ops.quantize_rows(torch.randn(rows, k, device="cuda"))
    want = ops._int8_product(x, weight, torch.float32, pair=pair, tile=8)

    def call():
        return ops._int8_product(x, weight, torch.float32, pair=pair)

    assert torch.equal(call(), want) and torch.equal(call(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(call(), want) and torch.equal(out, want)


def test_split_products_on_two_streams(ops):
    made = []
    for i in range(2):
        weight = ops.quantize_weight(torch.randn(4096, 8192, device="cuda"))
        x = ops.quantize_rows(torch.randn(40, 8192, device="cuda"))
        made.append((x, weight, ops._int8_product(x, weight, torch.float32, tile=8), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for x, weight, want, stream in made:
            with torch.cuda.stream(stream):
                got.append((ops.linear(x, weight, torch.float32), want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)
