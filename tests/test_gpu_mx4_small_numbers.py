"""The 4-bit Linear on the GPU at the lower end of float32."""

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.mx4 import mx4_linear_forward, mx4_quantize
from tests.gpu_helpers import DEV, announce
from tests.mx4_checks import PARTS, STEP, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n", [(3, 128, 40), (40, 128, 2100), (150, 128, 2100), (300, 70, 8200), (1000, 256, 4224)])
@pytest.mark.parametrize("power", [-100, -109, -118, -126, -136])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_small_inputs(dtype, power, m, k, n):
    """The parts of a float32 are bf16 numbers, multiples of 2^-133: below 2^-109 its last bits are not all there."""
    announce(f"small inputs {dtype} {power} {m} {k} {n}")
    g = torch.Generator().manual_seed(m)
    w = mx4_quantize((torch.randn(n, k, generator=g) * 2.0 ** 100).to(DEV))
    x = (torch.randn(m, k, generator=g).double() * 2.0 ** power).float().to(dtype)
    y = mx4_linear_forward(x.to(DEV), w, dtype=torch.float32)
    values = ora.values(*w, k)
    ref, mag = ora.linear(x, values)
    bound = (PARTS[dtype] * k + 4) * STEP * mag + STEP * ref.abs()
    if dtype == torch.float32:
        bound = bound + 2.0 ** -133 * values.abs().sum(1)
    within(y, ref, bound, f"2^{power}")


@pytest.mark.parametrize("m,k,n", [(3, 128, 40), (40, 128, 2100), (300, 70, 8200), (1000, 256, 4224)])
@pytest.mark.parametrize("four", [False, True], ids=["floats", "4-bit"])
def test_small_weights(four, m, k, n):
    """Weights down to the format's smallest, 2^-128, which as a bf16 number is no normal one."""
    announce(f"small weights {four} {m} {k} {n}")
    g = torch.Generator().manual_seed(m)
    w = mx4_quantize((torch.randn(n, k, generator=g).double() * 2.0 ** -127).float().to(DEV))
    assert int((w[1] == 0).sum()) > 0 and bool((w[0] != 0).any())
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = (torch.randn(m, k, generator=g) * (2.0 ** 12 if dtype == torch.float16 else 2.0 ** 100)).to(dtype).to(DEV)
        given = mx4_quantize(x) if four else x
        y = mx4_linear_forward(given, w, dtype=torch.float32)
        ref, mag = ora.linear(ora.values(*given, k) if four else x, ora.values(*w, k))
        within(y, ref, (PARTS[dtype] * k + 4) * STEP * mag + STEP * ref.abs() + 3 * k * 2.0 ** -149, f"{dtype}")
