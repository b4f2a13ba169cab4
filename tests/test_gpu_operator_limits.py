"""GPU: the 4-bit layers, the RMSNorms and the rotary positions at their limits, against their definitions in 64 bits."""
import importlib
import math

import pytest
import torch

from test_gpu_operators import DEV, _gen

pytestmark = pytest.mark.gpu
PKG = "hunyuan3d-tools_b200"


@pytest.fixture(scope="module")
def rotary():
    return importlib.import_module(PKG + ".rotary")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,group,zeros", [(5, 256, 64, 64, True), (40, 256, 64, 64, False), (70, 1024, 272, 32, True),
                                               (300, 448, 144, 448, True), (300, 2048, 128, 128, False)])
def test_int4_infinite_activations_give_what_the_definition_gives(qu, dtype, m, k, n, group, zeros):
    """For few rows and for many: an infinity keeps the weight's sign, two that cancel and a weight of zero give NaN, and the
    other rows stay as they are."""
    g = _gen(m + k)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV)
    zero = torch.randint(0, 16, (n, k // group), generator=g, device=DEV) if zeros else None
    scale = ((torch.rand(n, k // group, generator=g, device=DEV) - 0.5) * 0.02).to(dtype)      # of both signs
    layer = qu.Int4Linear.from_codes(codes, scale, zero)
    x = torch.randn(m, k, generator=g, device=DEV).to(dtype)
    x[0, 3], x[1, k - 1], x[2, 5], x[2, k // 2], x[3, 0], x[m - 1, 77] = math.inf, -math.inf, math.inf, math.inf, math.nan, math.inf
    y, ref = layer(x), x.double() @ layer.dequantize_weight().double().t()
    bad = ~ref.isfinite()
    assert torch.equal(~y.isfinite(), bad) and bool(ref[0].isinf().any()) and bool(ref[0].isnan().any())
    assert torch.equal(y[bad].isnan(), ref[bad].isnan())
    assert torch.equal(y[bad & ~ref.isnan()].double(), ref[bad & ~ref.isnan()])
