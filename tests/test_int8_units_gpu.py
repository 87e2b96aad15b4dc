"""Gate/up products in 8 bits: a row's results do not depend on the rows beside it."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_device):
    from tokensprint_amd.kernels import load_hip_ops
    return load_hip_ops(gpu_device)


UNITS = [{}, {"limit": 1.5}, {"act": "gelu_tanh"}]


@pytest.mark.parametrize("unit", UNITS)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_the_same_bits_in_every_tile(ops, gpu_device, unit, out_dtype):
    g = torch.Generator().manual_seed(3)
    rows = ops.quantize_rows(torch.randn(70, 1100, generator=g).to(gpu_device))
    weight = ops.quantize_weight((0.1 * torch.randn(2 * 200, 1100, generator=g)).to(gpu_device))
    limit = ops._unit(unit.get("limit"), unit.get("act", "silu"))
    want = ops._int8_product(rows, weight, out_dtype, pair=True, unit=limit, tile=9)
    for tile in range(9):
        assert torch.equal(ops._int8_product(rows, weight, out_dtype, pair=True, unit=limit, tile=tile), want), tile


@pytest.mark.parametrize("unit", UNITS)
def test_the_same_bits_beside_any_number_of_rows(ops, gpu_device, unit):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(300, 1024, generator=g).to(gpu_device).bfloat16()
    weight = ops.quantize_weight((0.1 * torch.randn(2 * 640, 1024, generator=g)).to(gpu_device))
    want = ops.linear_silu_mul(x, weight, torch.float32, **unit)
    for rows in (1, 2, 5, 17, 64, 129):
        assert torch.equal(ops.linear_silu_mul(x[:rows].contiguous(), weight, torch.float32, **unit), want[:rows]), rows


@pytest.mark.parametrize("unit", UNITS)
@pytest.mark.parametrize("rows", [1, 3, 20, 100, 300])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_is_no_number_stays_so(ops, gpu_device, unit, rows, value):
    """A row, or an output channel, with a NaN or an infinity gives NaN behind every unit, clamped ones too; the
    others know nothing of it."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(rows, 640, generator=g).to(gpu_device)
    w = (0.1 * torch.randn(2 * 96, 640, generator=g)).to(gpu_device)
    want = ops.linear_silu_mul(x, ops.quantize_weight(w), torch.float32, **unit)
    assert torch.isfinite(want).all()
    bad = x.clone()
    bad[rows // 2, 77] = value
    got = ops.linear_silu_mul(bad, ops.quantize_weight(w), torch.float32, **unit)
    keep = torch.arange(rows, device=gpu_device) != rows // 2
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[rows // 2]).all()
    assert torch.isnan(ops.linear(bad, ops.quantize_weight(w), torch.float32)[rows // 2]).all()
    for channel in (5, 96 + 5):                       # of the gate, of the up rows
        weight = w.clone()
        weight[channel, 33] = value
        got = ops.linear_silu_mul(x, ops.quantize_weight(weight), torch.float32, **unit)
        others = torch.arange(96, device=gpu_device) != 5
        assert torch.equal(got[:, others], want[:, others]) and torch.isnan(got[:, 5]).all()


@pytest.mark.parametrize("unit", UNITS)
@pytest.mark.parametrize("rows", [1, 3, 20, 100, 300])
def test_gates_whose_square_is_no_float32(ops, gpu_device, unit, rows):
    """Gates of some 1e20 are finite, and so is what the unit makes of them: the unit's weight is 0 or 1 there."""
    g = torch.Generator().manual_seed(6)
    x = (4e19 * torch.randn(rows, 640, generator=g)).to(gpu_device)
    gate, up = torch.randn(96, 640, generator=g), 1e-20 * torch.randn(96, 640, generator=g)
    weight = ops.quantize_weight(torch.cat([gate, up]).to(gpu_device))
    held = ops.quantize_rows(x)
    sums = held.codes.double().cpu() @ weight.codes.double().cpu().T
    y = sums * held.scales.double().cpu()[:, None] * weight.scales.double().cpu()
    big, u = y[:, :96], y[:, 96:]
    assert big.abs().max() > 2e19 and (big.abs() > 1e5).all()
    if "limit" in unit:
        want = torch.where(big > 0, 1.5 * torch.sigmoid(torch.tensor(1.5 * 1.702).double()), 0.0) * (u.clamp(-1.5, 1.5) + 1)
    else:
        want = big.clamp(min=0) * u
    got = ops.linear_silu_mul(x, weight, torch.float32, **unit).double().cpu()
    # two roundings for each of the two products' results, an ulp each of exp2 and reciprocal (and half a one of its
    # argument, 3.7 at the most in units of log2, times ln 2), the sums and products of the unit: below 16 halves of an ulp;
    # where u + 1 cancels, u's share of that
    bound = 2.0 ** -20 * (want.abs() + torch.where(big > 0, 2.0, 0.0)) if "limit" in unit else 2.0 ** -20 * want.abs()
    assert bool(((got - want).abs() <= bound).all())
