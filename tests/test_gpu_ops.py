"""The operators at a model's two ends against plain 64-bit computations.

Every tolerance is a bound on the operator's own roundings, element by element:
``U[dtype]`` is the largest relative error of one rounding to that type, and an fp32
sum over a chain of k adds is off by at most k * 2^-24 times the sum of its terms'
sizes.
"""
from __future__ import annotations

import math

import pytest
import torch

from slideformer_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -149}     # half the smallest number
U32 = 2.0 ** -24


def _gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def _normal(gen, device, *shape):
    return torch.randn(*shape, generator=gen, device=device)


def _within(got, want, bound, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(off[bad].max()), float((off / bound.clamp(min=1e-300)).max()))


def _strided(t, gap=0, offset=0):
    """The same matrix with rows `gap` elements apart, `offset` elements into its memory."""
    if t.dim() == 1:
        buf = torch.full((t.numel() + offset,), float("nan"), dtype=t.dtype, device=t.device)
        buf[offset:] = t
        return buf[offset:]
    n, h = t.shape
    buf = torch.full((offset + n * (h + gap),), float("nan"), dtype=t.dtype, device=t.device)
    view = buf[offset:].view(n, h + gap)[:, :h]
    view.copy_(t)
    return view


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,vocab,hidden,gap,offset,token", [
    (1, 7, 1, 0, 0, torch.int64), (1, 1000, 4096, 0, 0, torch.int32), (37, 50, 63, 0, 0, torch.int64),
    (129, 1000, 1023, 2, 1, torch.int64), (500, 300, 768, 8, 3, torch.int32), (64, 9, 5001, 0, 0, torch.int64)])
def test_embedding_is_the_rounded_product(hip_device, dtype, n, vocab, hidden, gap, offset, token):
    gen = _gen(hip_device, n + hidden)
    weight = _strided(_normal(gen, hip_device, vocab, hidden).to(dtype), gap, offset)
    tokens = torch.randint(0, vocab, (n,), generator=gen, device=hip_device).to(token)
    for scale in (1.0, math.sqrt(hidden)):
        got = ops.embedding(tokens, weight, scale=scale)
        want = (weight[tokens.long()].float() * torch.tensor(scale, dtype=F32)).to(dtype)   # one IEEE product
        assert torch.equal(got, want)
    out = _strided(torch.zeros(n, hidden, dtype=dtype, device=hip_device), 4, 1)
    assert ops.embedding(tokens, weight, out=out) is out
    assert torch.equal(out, weight[tokens.long()])
    assert ops.embedding(tokens.view(1, n, 1), weight).shape == (1, n, 1, hidden)


def test_embedding_of_bad_and_no_tokens(hip_device):
    weight = torch.ones(5, 33, dtype=BF16, device=hip_device)
    tokens = torch.tensor([0, -1, 5, 4, 1 << 40], device=hip_device)
    got = ops.embedding(tokens, weight)
    assert torch.equal(got.isnan().all(1).cpu(), torch.tensor([False, True, True, False, True]))
    assert bool((got[[0, 3]] == 1).all())
    assert ops.embedding(tokens[:0], weight).shape == (0, 33)


def _embedding_grad_exact(tokens, grad, vocab, scale):
    """(gradient, sum of sizes, count) per row, in 64 bits."""
    ok = (tokens >= 0) & (tokens < vocab)
    t, g = tokens[ok].long(), grad[ok].double()
    shape = (vocab, grad.shape[1])
    total = torch.zeros(shape, dtype=torch.float64, device=grad.device).index_add_(0, t, g) * scale
    sizes = torch.zeros(shape, dtype=torch.float64, device=grad.device).index_add_(0, t, g.abs()) * abs(scale)
    return total, sizes, torch.bincount(t, minlength=vocab)[:, None]


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("n,vocab,hidden,spread,gap", [
    (1, 3, 7, 3, 0), (15, 40, 64, 5, 0), (16, 40, 65, 1, 3), (17, 4, 513, 4, 0), (300, 1000, 1023, 2, 1),
    (4096, 500, 40, 500, 0), (4097, 70000, 24, 70000, 0), (9000, 5000, 136, 30, 8), (20000, 8, 16, 8, 0)])
def test_embedding_grad(hip_device, dtype, out_dtype, n, vocab, hidden, spread, gap):
    gen = _gen(hip_device, n + vocab)
    tokens = torch.randint(0, spread, (n,), generator=gen, device=hip_device)
    grad = _strided(_normal(gen, hip_device, n, hidden).to(dtype), gap)
    scale = 1.75
    want, sizes, count = _embedding_grad_exact(tokens, grad, vocab, scale)
    got = torch.full((vocab, hidden + gap), float("nan"), dtype=out_dtype, device=hip_device)[:, :hidden]
    ops.embedding_grad(tokens, grad, got, scale=scale)
    # the sum's chain is no longer than its terms, then the scale's product
    bound = U[out_dtype] * want.abs() + (count + 2) * U32 * sizes + TINY[out_dtype]
    _within(got, want, bound)
    assert bool((got[(count == 0).flatten()] == 0).all())
    again = torch.empty(vocab, hidden, dtype=out_dtype, device=hip_device)
    ops.embedding_grad(tokens.int(), grad, again, scale=scale)
    assert torch.equal(got, again)                           # a fixed order: equal bits, any layout
    # on top of what is there
    base = _normal(gen, hip_device, vocab, hidden).to(out_dtype)
    added = base.clone()
    ops.embedding_grad(tokens, grad, added, scale=scale, accumulate=True)
    total = want + base.double()
    _within(added, total, U[out_dtype] * total.abs() + (count + 3) * U32 * (sizes + base.double().abs()) +
            TINY[out_dtype])
    untouched = (count == 0).flatten()
    assert torch.equal(added[untouched], base[untouched])


def test_embedding_grad_leaves_out_padding_and_bad_tokens(hip_device):
    gen = _gen(hip_device, 5)
    tokens = torch.randint(-2, 12, (5000,), generator=gen, device=hip_device)
    grad = _normal(gen, hip_device, 5000, 96)
    got = ops.embedding_grad(tokens, grad, torch.empty(10, 96, device=hip_device), padding_idx=3)
    want, sizes, count = _embedding_grad_exact(tokens, grad, 10, 1.0)
    want[3], sizes[3] = 0, 0
    _within(got, want, (count + 3) * U32 * sizes + TINY[F32])
    # NaN in rows that take no part reaches nothing
    grad[(tokens == 3) | (tokens < 0) | (tokens > 9)] = float("nan")
    assert torch.equal(ops.embedding_grad(tokens, grad, torch.empty(10, 96, device=hip_device), padding_idx=3), got)
    nothing = ops.embedding_grad(tokens[:0], grad[:0], torch.full((10, 96), 2.0, device=hip_device))
    assert bool((nothing == 0).all())


def test_embedding_grad_is_the_difference_quotient(hip_device):
    """sum(c * embedding(W)) is linear in W: its difference along a direction is the gradient's product with it."""
    gen = _gen(hip_device, 6)
    tokens = torch.randint(0, 40, (200,), generator=gen, device=hip_device)
    weight, along = (_normal(gen, hip_device, 40, 31) for _ in range(2))
    c = _normal(gen, hip_device, 200, 31)
    grad = ops.embedding_grad(tokens, c, torch.empty_like(weight), scale=2.0)
    diff = sum(s * (ops.embedding(tokens, weight + s * 0.5 * along, scale=2.0).double() * c.double()).sum()
               for s in (1, -1))
    assert abs(float(diff - (grad.double() * along.double()).sum())) < 1e-5 * 200 * 31


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------
def _chain(hidden):
    """Adds a term of a row's sum goes through at most: a thread's own, then the tree over threads."""
    return max(64, hidden // 200) + 16


NORM_SIZES = [(1, 1), (3, 7), (1, 4096), (5, 64), (7, 513), (33, 1023), (6, 1024), (9, 2056), (4, 5120), (3, 8192),
              (2, 12289), (2, 16384), (3, 20001)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,hidden", NORM_SIZES)
@pytest.mark.parametrize("with_residual,gap", [(True, 0), (False, 3)])
def test_rms_norm(hip_device, dtype, n, hidden, with_residual, gap):
    gen = _gen(hip_device, n * hidden)
    x = _strided(_normal(gen, hip_device, n, hidden).to(dtype), gap, gap)
    residual = _strided((_normal(gen, hip_device, n, hidden) * 3).to(dtype), gap) if with_residual else None
    weight = (1 + _normal(gen, hip_device, hidden) * 0.2).to(dtype)
    eps = 1e-5
    out, summed, rstd = ops.rms_norm(x, weight, eps=eps, residual=residual)
    z = x.double() + (residual.double() if with_residual else 0)
    r = (z.square().mean(1) + eps).rsqrt()
    want = z * r[:, None] * weight.double()
    if with_residual:
        _within(summed, z, U[dtype] * z.abs() + U32 * z.abs() + TINY[dtype], "sum")
    else:
        assert summed is x
    # the sum of squares carries its chain's error, halved by the root; then mean, eps, root, quotient
    off = (_chain(hidden) / 2 + 6) * U32
    _within(rstd, r, off * r, "rstd")
    _within(out, want, (U[dtype] + off + 4 * U32) * want.abs() + TINY[dtype], "out")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,hidden", NORM_SIZES)
@pytest.mark.parametrize("eight", [torch.int8, torch.float8_e4m3fn])
def test_rms_norm_8bit(hip_device, dtype, n, hidden, eight):
    gen = _gen(hip_device, n * hidden + 1)
    x = _normal(gen, hip_device, n, hidden).to(dtype)
    residual = _normal(gen, hip_device, n, hidden).to(dtype)
    weight = (1 + _normal(gen, hip_device, hidden) * 0.2).to(dtype)
    out, scales, summed = ops.rms_norm_8bit(x, weight, eps=1e-5, residual=residual, dtype=eight)
    z = x.double() + residual.double()
    want = z * (z.square().mean(1) + 1e-5).rsqrt()[:, None] * weight.double()
    top = 127 if eight == torch.int8 else 448
    off = (_chain(hidden) / 2 + 10) * U32
    _within(scales, want.abs().amax(1) / top, (off + 2 * U32) * want.abs().amax(1) / top, "scales")
    # int8: half a step; fp8 with 3 bits of mantissa: 2^-4 of the value, or half the smallest step 2^-9
    step = scales.double()[:, None] * torch.ones_like(want)
    bound = 0.5 * step if eight == torch.int8 else torch.maximum(want.abs() * 2.0 ** -4, step * 2.0 ** -10)
    _within(out.double() * scales.double()[:, None], want, bound + 4 * off * want.abs().amax(1)[:, None] + 1e-30)
    _within(summed, z, (U[dtype] + U32) * z.abs() + TINY[dtype], "sum")


def test_rms_norm_of_zeros_infinities_and_nothing(hip_device):
    x = torch.ones(5, 96, dtype=BF16, device=hip_device)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 90] = float("nan")
    weight = torch.ones(96, dtype=BF16, device=hip_device)
    out, _, rstd = ops.rms_norm(x, weight, eps=0.5)
    assert bool((out[1] == 0).all()) and bool(out[3].isnan().all())
    assert bool(out[2, 5].isnan()) and float(rstd[2]) == 0.0
    assert bool((out[[0, 4]] - 1.5 ** -0.5).abs().max() < 2.0 ** -8)
    for eight in (torch.int8, torch.float8_e4m3fn):
        q, scales, _ = ops.rms_norm_8bit(x, weight, eps=0.5, dtype=eight)
        assert float(scales[1]) == 0.0 and bool(scales[[2, 3]].isnan().all())
        assert bool((q[[1, 2, 3]].float() == 0).all())
        assert bool((q[[0, 4]].float() == (127 if eight == torch.int8 else 448)).all())
    out, z, rstd = ops.rms_norm(x[:0], weight)
    assert out.shape == (0, 96) and rstd.shape == (0,)


@pytest.mark.parametrize("dtype,w_dtype", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("n,hidden", NORM_SIZES + [(700, 64), (1100, 515), (1500, 2048)])
@pytest.mark.parametrize("past,gap", [(True, 0), (False, 5)])
def test_rms_norm_grad(hip_device, dtype, w_dtype, n, hidden, past, gap):
    gen = _gen(hip_device, n + hidden)
    summed = _strided(_normal(gen, hip_device, n, hidden).to(dtype), gap)
    grad_out = _strided(_normal(gen, hip_device, n, hidden).to(dtype), gap, gap)
    grad_past = _normal(gen, hip_device, n, hidden).to(dtype) if past else None
    weight = (1 + _normal(gen, hip_device, hidden) * 0.2).to(dtype)
    rstd = (summed.float().square().mean(1) + 1e-5).rsqrt()
    r = rstd.double()[:, None]
    u, g = summed.double() * r, grad_out.double() * weight.double()
    inner = (g * u).mean(1, keepdim=True)
    want = (g - u * inner) * r + (grad_past.double() if past else 0)
    before = _normal(gen, hip_device, hidden).to(w_dtype)
    grad_x, grad_weight = ops.rms_norm_grad(grad_out, summed, rstd, weight, grad_summed=grad_past,
                                            grad_weight=torch.full_like(before, float("nan")))
    sizes = (g.abs() + u.abs() * (g * u).abs().mean(1, keepdim=True)) * r + (grad_past.double().abs() if past else 0)
    _within(grad_x, want, U[dtype] * want.abs() + (_chain(hidden) + 12) * U32 * sizes + TINY[dtype], "grad_x")
    total, size = (grad_out.double() * u).sum(0), (grad_out.double() * u).abs().sum(0)
    chain = n / 512 + 64
    _within(grad_weight, total, U[w_dtype] * total.abs() + (chain + 4) * U32 * size + TINY[w_dtype], "grad_weight")
    added = before.clone()
    again, added = ops.rms_norm_grad(grad_out, summed, rstd, weight, grad_summed=grad_past, grad_weight=added,
                                     accumulate=True)
    assert torch.equal(again, grad_x)
    total, size = total + before.double(), size + before.double().abs()
    _within(added, total, U[w_dtype] * total.abs() + (chain + 5) * U32 * size + TINY[w_dtype], "accumulated")


def test_rms_norm_grad_is_the_difference_quotient(hip_device):
    """fp32, central differences of sum(c * rms_norm): their own error is of third order in the step."""
    gen = _gen(hip_device, 9)
    z, c, along = (_normal(gen, hip_device, 5, 301) for _ in range(3))
    weight, weight_along = _normal(gen, hip_device, 301), _normal(gen, hip_device, 301)
    out, summed, rstd = ops.rms_norm(z, weight, eps=1e-5)
    grad_x, grad_weight = ops.rms_norm_grad(c, summed, rstd, weight)
    step = 1e-2

    def value(s, t):
        y = ops.rms_norm(z + s * along, weight + t * weight_along, eps=1e-5)[0]
        return float((y.double() * c.double()).sum())

    slope = (value(step, 0) - value(-step, 0)) / (2 * step)
    assert abs(slope - float((grad_x.double() * along.double()).sum())) < 2e-2
    slope = (value(0, step) - value(0, -step)) / (2 * step)
    assert abs(slope - float((grad_weight.double() * weight_along.double()).sum())) < 2e-2


def test_rms_norm_grad_of_no_rows(hip_device):
    none = torch.empty(0, 64, dtype=BF16, device=hip_device)
    weight = torch.ones(64, dtype=BF16, device=hip_device)
    grad_x, grad_weight = ops.rms_norm_grad(none, none, torch.empty(0, device=hip_device), weight)
    assert grad_x.shape == (0, 64) and bool((grad_weight == 0).all())


# ---------------------------------------------------------------------------
# loss
# ---------------------------------------------------------------------------
IGNORE = -100


def _loss_inputs(device, n, hidden, vocab, dtype, ignored, seed=0, gap=0, offset=0):
    gen = _gen(device, n + hidden + vocab + seed)
    x = _strided(_normal(gen, device, n, hidden).to(dtype), gap, offset)
    weight = _strided((_normal(gen, device, vocab, hidden) * (2.0 / math.sqrt(hidden))).to(dtype), gap, offset)
    targets = torch.randint(0, vocab, (n,), generator=gen, device=device)
    targets[torch.rand(n, generator=gen, device=device) < ignored] = IGNORE
    return x, weight, targets


class _Exact:
    """Loss and gradients in 64 bits on `where`, with bounds on what the kernels' roundings may do."""

    def __init__(self, x, weight, targets, mean=True, scale=1.0, where="cpu"):
        u = U[x.dtype]
        self.where, self.dtype = where, x.dtype
        keep = (targets != IGNORE).to(where)
        x, w, t = x.double().to(where), weight.double().to(where), targets.to(where)
        x = torch.where(keep[:, None], x, torch.zeros_like(x))
        rows, at = torch.nonzero(keep).flatten(), t[keep]
        s = x[rows] @ w.t()
        lse = torch.logsumexp(s, 1)
        losses = torch.zeros(t.numel(), dtype=torch.float64, device=where)
        losses[rows] = lse - s[torch.arange(rows.numel(), device=where), at]
        # a score is an fp32 sum of hidden products; a few more roundings for exp and the sums over the vocabulary
        sizes = x[rows].abs() @ w.abs().t()
        score = (x.shape[1] + 64) * U32 * (sizes.amax(1) if rows.numel() else sizes.new_zeros(0))
        score = score + (s.abs().amax(1) if rows.numel() else score) * 8 * U32 + 64 * U32
        self.row_losses = losses
        self.row_bounds = torch.zeros_like(losses)
        self.row_bounds[rows] = 2 * score + 4 * U32 * losses[rows].abs()
        count = max(1, rows.numel()) if mean else 1
        self.loss = losses.sum() / count
        self.loss_bound = self.row_bounds.sum() / count + 4 * U32 * self.loss.abs() + 1e-30
        p = torch.exp(s - lse[:, None])
        hot = torch.zeros_like(p)
        hot[torch.arange(rows.numel(), device=where), at] = 1
        f = scale / count
        # D: exp(s - m) rounded, its factor, D rounded; fp16 holds them times 2^13, steps of 2^-24 at the least
        d_off = p * (u + 4 * score[:, None] + 16 * U32) + (p + hot) * u + (2.0 ** -36 if self.dtype == F16 else 0)
        self.grad_x = torch.zeros_like(x)
        self.grad_x[rows] = (p - hot) @ w * f
        x_off = torch.zeros_like(x)
        chain = (w.shape[0] / 64 + 200) * U32
        x_off[rows] = (d_off + (p + hot) * chain) @ w.abs() * abs(f)
        self.grad_x_bound = x_off * 1.1 + u * self.grad_x.abs() + TINY[self.dtype]
        self.grad_w = (p - hot).t() @ x[rows] * f
        chain = (rows.numel() + 16) * U32
        self.grad_w_off = ((d_off + (p + hot) * chain).t() @ x[rows].abs()) * abs(f) * 1.1

    def check(self, loss, grad_x, grad_weight, before=None):
        _within(loss.to(self.where), self.loss, self.loss_bound, "loss")
        _within(grad_x.to(self.where), self.grad_x, self.grad_x_bound, "grad_x")
        want = self.grad_w + (0 if before is None else before.double().to(self.where))
        bound = self.grad_w_off + (U[grad_weight.dtype] + 4 * U32) * want.abs() + TINY[grad_weight.dtype]
        _within(grad_weight.to(self.where), want, bound, "grad_weight")


LOSS_SIZES = [
    # n, hidden, vocab, dtype, ignored
    (1, 64, 1, BF16, 0.0), (1, 1, 2, BF16, 0.0), (2, 8, 255, F16, 0.0), (13, 128, 1000, BF16, 0.0),
    (255, 192, 256, BF16, 0.3), (256, 256, 257, F16, 0.0), (257, 72, 513, BF16, 0.5), (300, 63, 700, BF16, 0.2),
    (515, 1023, 2003, F16, 0.5), (600, 320, 5000, BF16, 0.9), (1030, 64, 300, BF16, 0.1), (64, 1088, 3001, BF16, 0.0),
]


@pytest.mark.parametrize("n,hidden,vocab,dtype,ignored", LOSS_SIZES)
def test_linear_cross_entropy(hip_device, n, hidden, vocab, dtype, ignored):
    x, weight, targets = _loss_inputs(hip_device, n, hidden, vocab, dtype, ignored)
    e = _Exact(x, weight, targets)
    rows = ops.linear_cross_entropy(x, weight, targets, reduction="none")
    _within(rows.cpu(), e.row_losses, e.row_bounds + 1e-30, "rows")
    _within(ops.linear_cross_entropy(x, weight, targets).cpu(), e.loss, e.loss_bound, "mean")
    _within(ops.linear_cross_entropy(x, weight, targets, reduction="sum").cpu(), e.row_losses.sum(),
            e.row_bounds.sum() + 4 * U32 * e.row_losses.sum() + 1e-30, "sum")


@pytest.mark.parametrize("n,hidden,vocab,dtype,ignored", LOSS_SIZES)
def test_linear_cross_entropy_grad(hip_device, n, hidden, vocab, dtype, ignored):
    x, weight, targets = _loss_inputs(hip_device, n, hidden, vocab, dtype, ignored)
    e = _Exact(x, weight, targets)
    got = ops.linear_cross_entropy_grad(x, weight, targets)
    e.check(*got)
    again = ops.linear_cross_entropy_grad(x, weight, targets)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype,ignored", [(BF16, 0.0), (F16, 0.03)])
def test_linear_cross_entropy_grad_of_a_batch(hip_device, dtype, ignored):
    """Large enough that all three products take the larger tiles, and the states' gradient is split."""
    x, weight, targets = _loss_inputs(hip_device, 2040, 2048, 32700, dtype, ignored)
    e = _Exact(x, weight, targets, where=hip_device)
    got = ops.linear_cross_entropy_grad(x, weight, targets)
    e.check(*got)
    in_pieces = ops.linear_cross_entropy_grad(x, weight, targets, piece_bytes=1 << 26)
    e.check(*in_pieces)
    _within(ops.linear_cross_entropy(x, weight, targets, reduction="none"), e.row_losses, e.row_bounds + 1e-30)


@pytest.mark.parametrize("n,ignored", [(1030, 0.1), (1030, 0.8), (600, 0.0), (1030, 1.0)])
def test_linear_cross_entropy_in_pieces_and_on_top(hip_device, n, ignored):
    """Pieces of 256 rows, of which none, some or most are empty; grads of either type, added to what is there;
    a factor from the device; rows of every tensor further apart than they are long."""
    for dtype, w_dtype in ((BF16, BF16), (F16, F32)):
        x, weight, targets = _loss_inputs(hip_device, n, 128, 999, dtype, ignored, gap=8, offset=8)
        scale = torch.tensor(0.75, device=hip_device)
        gen = _gen(hip_device, 3)
        before = (_normal(gen, hip_device, 999, 128) * 1e-2).to(w_dtype)
        for reduction in ("mean", "sum"):
            e = _Exact(x, weight, targets, reduction == "mean", 0.75)
            target = _strided(before, 3, 1)
            got = ops.linear_cross_entropy_grad(x, weight, targets, reduction=reduction, grad_scale=scale,
                                                grad_weight=target, accumulate=True, piece_bytes=1)
            assert got[2] is target
            e.check(*got, before=before)
            fresh = torch.full_like(before, float("nan"))
            e.check(*ops.linear_cross_entropy_grad(x, weight, targets, reduction=reduction, grad_scale=scale,
                                                   grad_weight=fresh, piece_bytes=1))


def test_rows_without_a_target_reach_nothing(hip_device):
    x, weight, targets = _loss_inputs(hip_device, 400, 128, 777, BF16, 0.4)
    clean = ops.linear_cross_entropy_grad(x, weight, targets)
    x[targets == IGNORE] = float("nan")
    got = ops.linear_cross_entropy_grad(x, weight, targets)
    assert all(torch.equal(a, b) for a, b in zip(clean, got))
    assert bool((got[1][targets == IGNORE] == 0).all())
    # no row left: no loss and no gradient
    targets.fill_(IGNORE)
    loss, grad_x, grad_weight = ops.linear_cross_entropy_grad(x, weight, targets)
    assert float(loss) == 0.0 and not bool(grad_x.any()) and not bool(grad_weight.any())
    assert float(ops.linear_cross_entropy(x, weight, targets)) == 0.0
    # no row at all
    loss, grad_x, grad_weight = ops.linear_cross_entropy_grad(x[:0], weight, targets[:0])
    assert float(loss) == 0.0 and grad_x.shape == (0, 128) and not bool(grad_weight.any())
    assert ops.linear_cross_entropy(x[:0], weight, targets[:0], reduction="none").shape == (0,)
    # another index to ignore
    targets[:] = 5
    assert float(ops.linear_cross_entropy(x, weight, targets, ignore_index=5)) == 0.0


def test_bad_targets_and_infinite_scores_show(hip_device):
    x, weight, targets = _loss_inputs(hip_device, 300, 64, 500, BF16, 0.0)
    rows = ops.linear_cross_entropy(x, weight, targets, reduction="none")
    targets[7], targets[260] = 500, -3
    bad = torch.zeros(300, dtype=torch.bool, device=hip_device)
    bad[7] = bad[260] = True
    got = ops.linear_cross_entropy(x, weight, targets, reduction="none")
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], rows[~bad])
    loss, grad_x, _ = ops.linear_cross_entropy_grad(x, weight, targets)
    assert bool(loss.isnan()) and torch.equal(grad_x.isnan().any(1), bad)
    # a token whose scores are -inf for every state has no probability, and one of the lowest values hardly any
    x, weight, targets = _loss_inputs(hip_device, 300, 64, 500, BF16, 0.0)
    x[:, 0] = 1.0
    weight[:, 0] = 0.0
    keep = torch.ones(500, dtype=torch.bool)
    keep[[3, 499]] = False
    targets[(targets == 3) | (targets == 499)] = 4
    weight[3], weight[499] = 0, 0
    weight[3, 0], weight[499, 0] = float("-inf"), torch.finfo(BF16).min
    rows = ops.linear_cross_entropy(x, weight, targets, reduction="none")
    index = torch.cumsum(keep, 0).to(hip_device) - 1
    e = _Exact(x, weight[keep.to(hip_device)], index[targets])
    _within(rows.cpu(), e.row_losses, e.row_bounds + 1e-30)


def test_scores_far_from_zero(hip_device):
    """Scores of hundreds: the softmax is taken from the row's largest."""
    x, weight, targets = _loss_inputs(hip_device, 300, 64, 700, BF16, 0.0)
    x = (x.float() * 40).to(BF16)
    e = _Exact(x, weight, targets)
    e.check(*ops.linear_cross_entropy_grad(x, weight, targets))


def test_linear_cross_entropy_grad_is_the_difference_quotient(hip_device):
    """Central differences along directions that fp16 holds exactly; their own error is of third order."""
    x, weight, targets = _loss_inputs(hip_device, 40, 96, 350, F16, 0.25)
    gen = _gen(hip_device, 8)
    x, weight = (x * 16).round() / 16, (weight * 64).round() / 64
    _, grad_x, grad_weight = ops.linear_cross_entropy_grad(x, weight, targets, reduction="sum")
    for which, t, grad, step in (("x", x, grad_x, 1 / 32), ("weight", weight, grad_weight, 1 / 128)):
        along = torch.randint(-1, 2, t.shape, generator=gen, device=hip_device).to(F16)
        ends = [float(ops.linear_cross_entropy(t + s * step * along if which == "x" else x,
                                               weight if which == "x" else t + s * step * along, targets,
                                               reduction="sum")) for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * step)
        want = float((grad.double() * along.double()).sum())
        size = float((grad.double().square().sum().sqrt()))
        assert abs(slope - want) < 0.02 * size * math.sqrt(along.numel() / 40), (which, slope, want)


# ---------------------------------------------------------------------------
# all of them
# ---------------------------------------------------------------------------
def _all_outputs(x, residual, scales, weight, targets, tokens, stream=None):
    h = ops.embedding(tokens, weight, scale=2.0, stream=stream)
    out, summed, rstd = ops.rms_norm(x, scales, residual=residual, stream=stream)
    eight = ops.rms_norm_8bit(x, scales, residual=residual, stream=stream)
    loss, grad_x, grad_weight = ops.linear_cross_entropy_grad(out, weight, targets, stream=stream)
    grad_z, grad_scales = ops.rms_norm_grad(grad_x, summed, rstd, scales, stream=stream)
    ops.embedding_grad(targets, grad_z, grad_weight, accumulate=True, stream=stream)
    rows = ops.linear_cross_entropy(out, weight, targets, reduction="none", stream=stream)
    return [h, out, summed, rstd, *eight, loss, grad_x, grad_z, grad_scales, grad_weight, rows]


def test_calls_run_on_the_stream_they_are_given(hip_device):
    x, weight, targets = _loss_inputs(hip_device, 700, 192, 900, BF16, 0.2)
    residual = torch.flip(x, (0,)).contiguous()
    scales = torch.linspace(0.5, 1.5, 192, device=hip_device).to(BF16)
    tokens = targets.clamp(min=0)
    want = _all_outputs(x, residual, scales, weight, targets, tokens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(hip_device)
    late = [torch.zeros_like(t) for t in (x, residual, scales, weight)]
    late_targets, late_tokens = torch.full_like(targets, IGNORE), torch.zeros_like(tokens)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                        # the inputs come late on the side stream
        for to, t in zip(late, (x, residual, scales, weight)):
            to.copy_(t)
        late_targets.copy_(targets)
        late_tokens.copy_(tokens)
    got = _all_outputs(*late, late_targets, late_tokens, stream=side)
    with torch.cuda.stream(side):
        again = _all_outputs(*late, late_targets, late_tokens)
    raw = _all_outputs(*late, late_targets, late_tokens, stream=side.cuda_stream)
    side.synchronize()
    for other in (got, again, raw):
        assert all(torch.equal(a, b) for a, b in zip(want, other))


def test_calls_replay_in_a_graph(hip_device):
    x, weight, targets = _loss_inputs(hip_device, 300, 128, 600, BF16, 0.2)
    residual = torch.flip(x, (0,)).contiguous()
    scales = torch.linspace(0.5, 1.5, 128, device=hip_device).to(BF16)
    tokens = targets.clamp(min=0)
    _all_outputs(x, residual, scales, weight, targets, tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _all_outputs(x, residual, scales, weight, targets, tokens)
    for seed in range(3):
        x2, weight2, targets2 = _loss_inputs(hip_device, 300, 128, 600, BF16, 0.3, seed=seed)
        x.copy_(x2), weight.copy_(weight2), targets.copy_(targets2), residual.copy_(torch.flip(x2, (0,)))
        tokens.copy_(targets2.clamp(min=0))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = _all_outputs(x, residual, scales, weight, targets, tokens)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), seed


def test_python_refusals(hip_device):
    x, weight, targets = _loss_inputs(hip_device, 8, 64, 32, BF16, 0.0)
    scales = torch.ones(64, dtype=BF16, device=hip_device)
    rstd = torch.ones(8, device=hip_device)
    for match, call in (
            ("contiguous", lambda: ops.embedding(targets, weight.t())),
            ("dtype of tokens", lambda: ops.embedding(targets.float(), weight)),
            ("tokens on cpu", lambda: ops.embedding(targets.cpu(), weight)),
            ("size mismatch", lambda: ops.embedding(targets, weight, out=x[:4])),
            ("size mismatch", lambda: ops.embedding_grad(targets, x[:4], weight)),
            ("expected", lambda: ops.embedding_grad(targets, x, weight.to(F16))),
            ("size mismatch", lambda: ops.rms_norm(x, scales[:32])),
            ("dtype of weight", lambda: ops.rms_norm(x, scales.float())),
            ("residual is", lambda: ops.rms_norm(x, scales, residual=x.float())),
            ("contiguous", lambda: ops.rms_norm(x.t().contiguous().t(), scales)),
            ("size mismatch", lambda: ops.rms_norm_grad(x, x, rstd[:4], scales)),
            ("accumulate", lambda: ops.rms_norm_grad(x, x, rstd, scales, accumulate=True)),
            ("float32", lambda: ops.linear_cross_entropy(x.float(), weight.float(), targets)),
            ("x is", lambda: ops.linear_cross_entropy(x.to(F16), weight, targets)),
            ("dtype of targets", lambda: ops.linear_cross_entropy(x, weight, targets.int())),
            ("size mismatch", lambda: ops.linear_cross_entropy(x, weight, targets[:3])),
            ("empty", lambda: ops.linear_cross_entropy(x, weight[:0], targets)),
            ("accumulate", lambda: ops.linear_cross_entropy_grad(x, weight, targets, accumulate=True)),
            ("grad_weight is", lambda: ops.linear_cross_entropy_grad(x, weight, targets,
                                                                     grad_weight=weight.to(F16))),
            ("dtype of grad_scale", lambda: ops.linear_cross_entropy_grad(
                x, weight, targets, grad_scale=torch.ones((), dtype=torch.float64, device=hip_device)))):
        with pytest.raises(RuntimeError, match=match):
            call()
