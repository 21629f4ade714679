"""The loss of at most 16 rows over a large vocabulary, as a step of generation or a few held-out
tokens need it: the matrix is read where it lies, at any row distance and alignment."""
from __future__ import annotations

import pytest
import torch

from slideformer_amd import ops
from test_gpu_ops import BF16, F16, IGNORE, _Exact, _loss_inputs, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,ignored", [(1, 0.0), (13, 0.0), (16, 0.0), (16, 0.4), (17, 0.0)])
@pytest.mark.parametrize("vocab,hidden,gap,offset", [
    (65281, 1088, 0, 0), (65300, 1023, 0, 0), (70001, 1088, 8, 8), (70001, 1023, 2, 1), (65536, 257, 0, 3),
    (70001, 64, 0, 0), (65100, 1088, 0, 0), (65100, 1023, 4, 1)])
def test_few_rows_of_a_large_vocabulary(hip_device, dtype, n, ignored, vocab, hidden, gap, offset):
    x, weight, targets = _loss_inputs(hip_device, n, hidden, vocab, dtype, ignored, gap=gap, offset=offset)
    targets[0] = vocab - 1                                   # in the last tile, beside columns past the vocabulary
    e = _Exact(x, weight, targets, where=hip_device)
    rows = ops.linear_cross_entropy(x, weight, targets, reduction="none")
    _within(rows, e.row_losses, e.row_bounds + 1e-30, "rows")
    _within(ops.linear_cross_entropy(x, weight, targets), e.loss, e.loss_bound, "mean")
    got = ops.linear_cross_entropy_grad(x, weight, targets)
    e.check(*got)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.linear_cross_entropy_grad(x, weight, targets)))
    # rows that take no part may hold anything
    x[targets == IGNORE] = float("nan")
    assert torch.equal(ops.linear_cross_entropy(x, weight, targets, reduction="none"), rows)
