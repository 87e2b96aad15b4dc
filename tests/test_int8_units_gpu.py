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
