"""The state space operators without a GPU: workspaces, arguments that must not be
taken for others, tensors that overlap, modules in 16 bits."""

import pytest
import torch

from sparseflow_amd import _lib


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("each", [1, 16])
def test_a_scans_workspace_is_of_the_sequences_that_are_cut(dtype, each):
    """One long sequence among short ones: no workspace times the whole batch."""
    H, P, N, long, short = 64, 64, 128, 16384, 255
    tokens = long + short * each
    desc = _lib.scan_desc(short + 1, tokens, long, short + 1, *[(0, 1, 1)] * 5, H, P, 1, N, dtype, True)
    data = tokens * 2 * H * P * dtype.itemsize + 2 * (short + 1) * H * P * N * 4
    assert 0 < desc[2] < data // 4, f"{desc[2]} bytes of workspace for {data} of data"
