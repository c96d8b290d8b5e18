"""Scores that are all -infinity, on the GPU: few rows and many, whole and in parts of their tokens."""

import pytest
import torch

from tests.gpu_helpers import DEV, announce
from tests.mx4_score_checks import check_scores_of_minus_infinity

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,old", [(1, 0), (1, 40), (3, 5000), (60, 40), (130, 0), (60, 4000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_scores_of_minus_infinity(dtype, n, old):
    announce(f"scores of -inf {dtype} {n} {old}")
    check_scores_of_minus_infinity(DEV, dtype, n, old)
