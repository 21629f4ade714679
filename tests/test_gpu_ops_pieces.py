"""The loss with its gradients over several pieces of rows, at sizes of whole batches,
against 64 bits on the device."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from slideformer_amd import _lib, _ops_lib, ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -149}
U32 = 2.0 ** -24
IGNORE = -100


def _exact(x, weight, targets, scale):
    """(loss, its bound, grad_x, its bound, grad_weight, the bound of its sum before it is rounded)."""
    u, keep = U[x.dtype], torch.nonzero(targets != IGNORE).flatten()
    xs, w, at = x[keep].double(), weight.double(), targets[keep]
    rows = torch.arange(keep.numel(), device=x.device)
    s = xs @ w.t()
    lse = torch.logsumexp(s, 1)
    losses = lse - s[rows, at]
    # a score is an fp32 sum of hidden products; a few more roundings for exp and the sums over the vocabulary
    score = (x.shape[1] + 64) * U32 * (xs.abs() @ w.abs().t()).amax(1) + 8 * U32 * s.abs().amax(1) + 64 * U32
    p = torch.exp(s - lse[:, None])
    hot = torch.zeros_like(p)
    hot[rows, at] = 1
    f = scale / max(1, keep.numel())
    # D: exp(s - m) rounded, its factor, D rounded; fp16 holds them times 2^13, steps of 2^-24 at the least
    off = p * (u + 4 * score[:, None] + 16 * U32) + (p + hot) * u + (2.0 ** -36 if x.dtype == F16 else 0)
    grad_x, x_bound = (torch.zeros(x.shape, dtype=torch.float64, device=x.device) for _ in range(2))
    grad_x[keep] = (p - hot) @ w * f
    x_bound[keep] = (off + (p + hot) * ((w.shape[0] / 64 + 200) * U32)) @ w.abs() * f * 1.1
    x_bound += u * grad_x.abs() + TINY[x.dtype]
    grad_w = (p - hot).t().contiguous() @ xs * f
    w_off = (off + (p + hot) * ((keep.numel() + 16) * U32)).t().contiguous() @ xs.abs() * f * 1.1
    count = max(1, keep.numel())
    return (losses.sum() / count, (2 * score + 4 * U32 * losses.abs()).sum() / count + 4 * U32 * losses.sum() / count,
            grad_x, x_bound, grad_w, w_off)


@pytest.mark.parametrize("dtype,w_dtype", [(BF16, BF16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("n,hidden,vocab,ignored,pieces", [
    (2040, 512, 32700, 0.0, 2), (2040, 512, 32700, 0.6, 2), (3100, 200, 20100, 0.1, 5), (1500, 1023, 8001, 0.0, 4)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_pieces_of_a_batch(hip_device, dtype, w_dtype, n, hidden, vocab, ignored, pieces, accumulate):
    gen = torch.Generator(device=hip_device).manual_seed(n + hidden + vocab)
    x = torch.randn(n, hidden, generator=gen, device=hip_device).to(dtype)
    weight = (torch.randn(vocab, hidden, generator=gen, device=hip_device) * (2 / math.sqrt(hidden))).to(dtype)
    targets = torch.randint(0, vocab, (n,), generator=gen, device=hip_device)
    targets[torch.rand(n, generator=gen, device=hip_device) < ignored] = IGNORE
    before = (torch.randn(vocab, hidden, generator=gen, device=hip_device) * 1e-2).to(w_dtype)
    given = before.clone() if accumulate else torch.full_like(before, float("nan"))
    scale = torch.tensor(0.75, device=hip_device)
    loss, grad_x, grad_weight = ops.linear_cross_entropy_grad(
        x, weight, targets, grad_scale=scale, grad_weight=given, accumulate=accumulate,
        piece_bytes=-(-n // pieces) * 2 * vocab)
    assert grad_weight is given
    want, bound, want_x, x_bound, want_w, w_off = _exact(x, weight, targets, 0.75)
    assert float((loss.double() - want).abs()) <= float(bound)
    assert not bool(((grad_x.double() - want_x).abs() > x_bound).any()) and not bool(grad_x.isnan().any())
    if accumulate:
        want_w += before.double()
    # the sum over pieces: an fp32 add for each, of sums of no more than the terms' sizes
    sizes = want_w.abs() + w_off / U[dtype] + (before.double().abs() if accumulate else 0)
    w_bound = w_off + U[w_dtype] * want_w.abs() + (pieces + 4) * U32 * sizes + TINY[w_dtype]
    assert not bool(((grad_weight.double() - want_w).abs() > w_bound).any()) and not bool(grad_weight.isnan().any())


def test_all_rows_through_the_c_abi(hip_device):
    """piece_rows 0: all rows, of which a launch takes 32768 at a time; the same bits as asked for in such pieces."""
    n, hidden, vocab = 70001, 64, 300
    gen = torch.Generator(device=hip_device).manual_seed(4)
    x = torch.randn(n, hidden, generator=gen, device=hip_device).to(BF16)
    weight = torch.randn(vocab, hidden, generator=gen, device=hip_device).to(BF16)
    targets = torch.randint(0, vocab, (n,), generator=gen, device=hip_device)
    lib, results = _ops_lib.load(), []
    for piece_rows in (0, 32768):
        loss = torch.empty((), device=hip_device)
        grad_x, grad_weight = torch.empty_like(x), torch.empty_like(weight)
        call = _ops_lib.LaLinearLoss(
            dtype=_lib.LA_BF16, x=x.data_ptr(), n=n, hidden=hidden, x_stride=hidden, weight=weight.data_ptr(),
            vocab=vocab, weight_stride=hidden, targets=targets.data_ptr(), ignore_index=IGNORE, mean=1,
            loss=loss.data_ptr(), grads=1, grad_x=grad_x.data_ptr(), grad_x_stride=hidden,
            grad_weight_dtype=_lib.LA_BF16, grad_weight=grad_weight.data_ptr(), grad_weight_stride=hidden,
            piece_rows=piece_rows)
        size = lib.la_linear_loss_workspace(ctypes.byref(call))
        work = torch.empty(size, dtype=torch.uint8, device=hip_device)
        stream = torch.cuda.current_stream(hip_device).cuda_stream
        assert lib.la_linear_loss(ctypes.byref(call), work.data_ptr(), size, stream) == _lib.LA_OK
        torch.cuda.synchronize()
        results.append((loss, grad_x, grad_weight))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    want, bound, want_x, x_bound, want_w, w_off = _exact(x, weight, targets, 1.0)
    assert float((results[0][0].double() - want).abs()) <= float(bound)
    assert not bool(((results[0][1].double() - want_x).abs() > x_bound).any())
    w_bound = w_off + U[BF16] * want_w.abs() + 8 * U32 * (want_w.abs() + w_off / U[BF16]) + TINY[BF16]
    assert not bool(((results[0][2].double() - want_w).abs() > w_bound).any())
