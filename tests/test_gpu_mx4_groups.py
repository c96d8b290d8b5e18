"""The 4-bit Linear of few tiles on the GPU: groups of wavefronts that add up what they have, many times over."""

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.mx4 import mx4_linear_forward, mx4_quantize
from tests.gpu_helpers import DEV, announce
from tests.mx4_checks import PARTS, STEP, half_step, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(128, 4096, 2048), (100, 2080, 4096), (250, 1056, 3000)])
def test_every_call_gives_the_same(m, k, n, dtype):
    """y has at most 256 tiles of 64 x 64 and is no few pieces.  The order of a sum's terms is fixed, so that calls agree to
    the bit, whatever else keeps the CUs busy."""
    announce(f"groups {m} {k} {n} {dtype}")
    g = torch.Generator().manual_seed(m)
    w = mx4_quantize((torch.randn(n, k, generator=g) * k ** -0.5).to(DEV))
    x = torch.randn(m, k, generator=g).to(dtype).to(DEV)
    y = mx4_linear_forward(x, w)
    ref, mag = ora.linear(x, ora.values(*w, k))
    within(y, ref, (PARTS[dtype] * k + 4) * STEP * mag + half_step(dtype) * ref.abs(), f"{m} {k} {n}")
    other = torch.cuda.Stream()
    busy = torch.randn(64 << 20, device=DEV)
    torch.cuda.synchronize()
    for turn in range(6):
        with torch.cuda.stream(other):
            for _ in range(4):
                busy.mul_(1.0)
        got = [mx4_linear_forward(x, w) for _ in range(20)]
        torch.cuda.synchronize()
        assert all(torch.equal(v, y) for v in got), turn
