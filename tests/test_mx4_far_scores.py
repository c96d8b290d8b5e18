"""Scores that are all -infinity, on the host: what the softmax of them is, and what a row without tokens is."""

import pytest
import torch

from tests.mx4_score_checks import check_scores_of_minus_infinity

CPU = torch.device("cpu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_scores_of_minus_infinity(dtype):
    check_scores_of_minus_infinity(CPU, dtype, 3, 40)
