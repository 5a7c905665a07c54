"""Layouts of the fine-tuning operators' operands: an adapter's factors, one long column."""
import pytest
import torch

import finetune_ref as R
from interior_amd import ops

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def rand(*shape, dtype=BF, scale=1.0, seed=0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def test_one_column_of_a_row_length_that_wraps(gpu):
    """K = 1 on 2^26 - 1 rows: copied to a padded row of 2^26 elements, 32 times whose bytes is 2^32; an infinity stays one."""
    m = 2 ** 26 - 1
    x, w = torch.ones(m, 1, dtype=BF, device=gpu), torch.tensor([[2.0], [-0.5], [1.0], [4.0], [0.25], [-1.0], [8.0], [0.5]], dtype=BF, device=gpu)
    x[5] = float("inf")
    assert torch.equal(ops.linear(x, w), x * w.t())  # powers of two: exact
