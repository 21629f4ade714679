"""The norm and rotation of heads and their gradient against plain 64-bit computations.

Tolerances are bounds on the operators' own roundings: ``U`` is one rounding to the type, ``U32`` one to
fp32.  A sum over dim elements is off by at most dim * U32 of its terms' sizes; 1 / sqrt(mean + eps) of
a sum of squares by (dim / 2 + 4) * U32, relative; a rotated element by 4 * U32 of its two products' sizes.
"""
from __future__ import annotations

import pytest
import torch

from slideformer_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -149}
U32 = 2.0 ** -24
EPS = 1e-5
NAN = float("nan")


def _within(got, want, bound, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(off[bad].max()), float((off / bound.clamp(min=1e-300)).max()))


def _pairs(rotated, interleaved):
    j = torch.arange(rotated // 2)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + rotated // 2)


def _turn(x, cos, sin, rotated, interleaved):
    a, b = (i.to(x.device) for i in _pairs(rotated, interleaved))
    y = x.clone()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


class Case:
    def __init__(self, device, dtype, n, heads, kv_heads, dim, rotated, interleaved=False, norms=(True, True), at=torch.int64,
                 lay=None, seed=0):
        gen = torch.Generator(device=device).manual_seed(seed + n + dim)

        def normal(std, *shape):
            return torch.randn(*shape, generator=gen, device=device).mul_(std)

        lay = lay or (lambda t: t)
        self.dtype, self.dim, self.rotated, self.interleaved = dtype, dim, rotated, interleaved
        self.x = [lay(normal(1.5, n, h, dim).to(dtype)) for h in (heads, kv_heads)]
        self.g = [lay(normal(1.0, n, h, dim).to(dtype)) for h in (heads, kv_heads)]
        self.w = [(1 + normal(0.3, dim)).to(dtype) if there else None for there in norms]
        angle = normal(2.0, 50, rotated // 2).double()
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        self.at = None if at is None else torch.randint(0, 50, (n,), generator=gen, device=device).to(at)
        rows = torch.arange(n, device=device) if at is None else self.at.long()
        self.c, self.s = (t.double()[rows][:, None] for t in (self.cos, self.sin))
        self.how = dict(q_weight=self.w[0], k_weight=self.w[1], positions=self.at, eps=EPS, interleaved=interleaved)

    def run(self, **more):
        return ops.qk_norm_rotary(*self.x, self.cos, self.sin, **self.how, **more)

    def grad(self, **more):
        return ops.qk_norm_rotary_grad(*self.g, *self.x, self.cos, self.sin, **self.how, **more)

    def turned(self, x, back=False):
        return _turn(x, self.c, -self.s if back else self.s, self.rotated, self.interleaved)

    def sizes(self, x):
        """The sizes of both products of a rotated element."""
        return _turn(x.abs(), self.c.abs(), -self.s.abs(), self.rotated, self.interleaved).abs() + \
            _turn(x.abs(), self.c.abs(), self.s.abs(), self.rotated, self.interleaved).abs()

    def check(self, got):
        u, tiny = U[self.dtype], TINY[self.dtype]
        for y, x, w in zip(got, self.x, self.w):
            x = x.double()
            if w is not None:
                x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
            want = self.turned(x)
            _within(y, want, u * want.abs() + (self.dim / 2 + 12) * U32 * self.sizes(x) + tiny, "out")

    def check_grads(self, got, kind=None):
        kind = kind or self.dtype
        tiny = TINY[self.dtype]
        for dx, dw, g, x, w in zip(got[:2], got[2:], self.g, self.x, self.w):
            turned = self.turned(g.double(), back=True)
            turned_off = 4 * U32 * self.sizes(g.double())
            if w is None:
                assert dw is None
                _within(dx, turned, U[self.dtype] * turned.abs() + turned_off + tiny, "grad without norm")
                continue
            x, w = x.double(), w.double()
            r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
            unit, gw = x * r, turned * w
            want = r * (gw - unit * (gw * unit).mean(-1, keepdim=True))
            rel = (self.dim / 2 + 8) * U32                   # of r
            gw_off = turned_off * w.abs() + U32 * gw.abs()
            mean_size = (gw * unit).abs().mean(-1, keepdim=True)
            mean_off = (gw_off * unit.abs()).mean(-1, keepdim=True) + (self.dim * U32 + 3 * rel) * mean_size
            off = r * (gw_off + unit.abs() * mean_off + (2 * rel + 4 * U32) * (gw.abs() + unit.abs() * mean_size))
            _within(dx, want, U[self.dtype] * want.abs() + (1 + U[self.dtype]) * off + tiny, "grad")
            terms = turned * unit
            total = terms.sum((0, 1))
            # each term, and chains of sums no longer than there are terms
            off = (turned_off * unit.abs() + (rel + 4 * U32) * terms.abs()).sum((0, 1)) + \
                min(terms[..., 0].numel(), 4096) * U32 * terms.abs().sum((0, 1))
            _within(dw, total, U[kind] * total.abs() + (1 + U[kind]) * off + TINY[kind], "grad of the scales")


SHAPES = [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (3, 4, 2, 64, 64), (37, 5, 1, 80, 40), (130, 2, 2, 96, 24), (17, 3, 1, 50, 50),
          (9, 4, 4, 63, 62), (700, 8, 2, 128, 128), (5, 2, 1, 256, 256), (11, 1, 1, 7, 0), (4097, 3, 1, 32, 16), (2, 0, 3, 16, 8)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,heads,kv_heads,dim,rotated", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_against_the_formula(hip_device, dtype, n, heads, kv_heads, dim, rotated, interleaved):
    case = Case(hip_device, dtype, n, heads, kv_heads, dim, rotated, interleaved)
    case.check(case.run())
    got = case.grad()
    case.check_grads(got)
    for a, b in zip(case.grad(), got):
        assert torch.equal(a, b)                             # a fixed order: equal bits


@pytest.mark.parametrize("norms", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("at", [None, torch.int32])
def test_without_norms_and_positions(hip_device, norms, at):
    case = Case(hip_device, BF16, 50, 6, 2, 128, 64, norms=norms, at=at)
    case.check(case.run())
    case.check_grads(case.grad())
    if norms == (False, False):
        # nothing of q and k is needed then
        got = ops.qk_norm_rotary_grad(*case.g, None, None, case.cos, case.sin, **case.how)
        case.check_grads(got)


def _fused(t):
    wide = torch.full((t.shape[0], t.shape[1] + 3, t.shape[2]), NAN, dtype=t.dtype, device=t.device)
    wide[:, 1:-2] = t
    return wide[:, 1:-2]


def _heads_first(t):
    return t.transpose(0, 1).contiguous().transpose(0, 1)


def _odd(t):
    n, h, d = t.shape
    buf = torch.full((n * (h * d + 1) + 1,), NAN, dtype=t.dtype, device=t.device)
    view = buf[1:].view(n, -1)[:, :-1].unflatten(1, (h, d))
    view.copy_(t)
    return view


@pytest.mark.parametrize("lay", [_fused, _heads_first, _odd])
@pytest.mark.parametrize("dtype,dim,rotated", [(BF16, 128, 128), (F32, 96, 50), (F16, 30, 20)])
def test_views_of_any_order_and_results_in_place(hip_device, lay, dtype, dim, rotated):
    case, plain = (Case(hip_device, dtype, 70, 6, 2, dim, rotated, lay=how) for how in (lay, None))
    want, want_grads = plain.run(), plain.grad()
    for a, b in zip(case.run(), want):
        assert torch.equal(a, b)
    for a, b in zip(case.grad(), want_grads):
        assert torch.equal(a, b)
    got = case.grad(out=tuple(case.g))
    assert got[0] is case.g[0] and got[1] is case.g[1]
    for a, b in zip(got, want_grads):
        assert torch.equal(a, b)
    got = case.run(out=tuple(case.x))
    assert got[0] is case.x[0]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_gradients_of_the_scales_on_top_of_others(hip_device):
    case = Case(hip_device, BF16, 300, 6, 2, 128, 128)
    fresh = case.grad(grad_q_weight=torch.empty(128, device=hip_device), grad_k_weight=torch.empty(128, device=hip_device))
    case.check_grads(fresh, F32)
    for kind in (BF16, F32):
        base = [torch.randn(128, device=hip_device).to(kind) for _ in range(2)]
        given = [b.clone() for b in base]
        got = case.grad(grad_q_weight=given[0], grad_k_weight=given[1], accumulate=True)
        for g, b, f in zip(got[2:], base, fresh[2:]):
            want = b.double() + f.double()
            _within(g, want, U[kind] * want.abs() + 4 * U32 * (b.double().abs() + f.double().abs()))
        assert got[2] is given[0]


def test_positions_outside_the_tables(hip_device):
    case = Case(hip_device, BF16, 4, 2, 1, 64, 32)
    case.at[:] = torch.tensor([3, -1, 50, 1 << 40], device=hip_device)
    for y in case.run():
        assert torch.equal(y[..., :32].isnan().all(-1).all(-1).cpu(), torch.tensor([False, True, True, True]))
        assert not bool(y[..., 32:].isnan().any())


def test_bad_elements_stay_in_their_head(hip_device):
    case = Case(hip_device, BF16, 20, 4, 2, 128, 64)
    want = case.run()
    case.x[0][3, 2, 100] = float("inf")
    case.x[1][5, 1, 3] = NAN
    got = case.run()
    bad = [torch.zeros(20, h, dtype=torch.bool, device=hip_device) for h in (4, 2)]
    bad[0][3, 2] = bad[1][5, 1] = True
    for g, w, b in zip(got, want, bad):
        assert torch.equal(g[~b], w[~b]) and bool(g[b].isnan().any())
    # without a norm, an infinity among the elements that do not turn stays alone
    case = Case(hip_device, BF16, 20, 4, 2, 128, 64, norms=(False, False))
    case.x[0][3, 2, 100] = float("inf")
    got = case.run()[0][3, 2]
    assert bool(got[100].isinf()) and bool(got[torch.arange(128, device=hip_device) != 100].isfinite().all())


def test_heads_of_zeros(hip_device):
    case = Case(hip_device, BF16, 5, 2, 1, 64, 64)
    for x in case.x:
        x.zero_()
    for y in case.run():
        assert bool((y == 0).all())
    case.check_grads(case.grad())


def test_distances_that_pass_32_bits(hip_device):
    n, step = 5000, 1 << 20
    buf = torch.empty(n * step, dtype=BF16, device=hip_device)
    case = Case(hip_device, BF16, n, 2, 1, 64, 64)
    want, want_grads = case.run(), case.grad()
    far = buf.as_strided((n, 2, 64), (step, 64, 1))
    far.copy_(case.x[0])
    case.x[0] = far
    for a, b in zip(case.run(out=(far.clone(), case.x[1].clone())), want):
        assert torch.equal(a, b)
    for a, b in zip(case.grad(), want_grads):
        assert torch.equal(a, b)


def test_gradient_is_the_difference_quotient(hip_device):
    case = Case(hip_device, F32, 30, 3, 2, 48, 32)
    got = case.grad()
    gen = torch.Generator(device=hip_device).manual_seed(3)

    def loss(q, k, wq, wk):
        total = 0.0
        for x, w, g in ((q, wq, case.g[0]), (k, wk, case.g[1])):
            y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
            total = total + (case.turned(y) * g.double()).sum()
        return float(total)

    base = [t.double() for t in (*case.x, *case.w)]
    for i, grad in enumerate(got):
        direction = torch.randn(grad.shape, generator=gen, device=hip_device, dtype=torch.float64)
        h = 1e-5
        ahead, back = ([t + sign * h * direction if j == i else t for j, t in enumerate(base)] for sign in (1, -1))
        slope = (loss(*ahead) - loss(*back)) / (2 * h)
        size = float((grad.double().abs() * direction.abs()).sum())
        assert abs(float((grad.double() * direction).sum()) - slope) < 1e-5 * size


def test_captured_and_replayed(hip_device):
    case = Case(hip_device, BF16, 200, 8, 2, 128, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        case.run(), case.grad()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = case.run(), case.grad()
    for step in range(4):
        gen = torch.Generator(device=hip_device).manual_seed(step)
        for t in (*case.x, *case.g):
            t.copy_(torch.randn(t.shape, generator=gen, device=hip_device))
        graph.replay()
        want, want_grads = case.run(), case.grad()
        torch.cuda.synchronize()
        for a, b in zip((*out, *grads), (*want, *want_grads)):
            assert torch.equal(a, b)


def test_on_another_stream_and_nothing_to_do(hip_device):
    case = Case(hip_device, BF16, 3000, 8, 2, 128, 128)
    want, want_grads = case.run(), case.grad()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, grads = case.run(stream=side), case.grad(stream=side)
    side.synchronize()
    for a, b in zip((*out, *grads), (*want, *want_grads)):
        assert torch.equal(a, b)
    none = Case(hip_device, BF16, 0, 4, 2, 64, 64)
    assert none.run()[0].shape == (0, 4, 64)
    got = none.grad()
    assert got[0].shape == (0, 4, 64) and bool((got[2] == 0).all()) and bool((got[3] == 0).all())
    base = torch.ones(64, dtype=BF16, device=hip_device)
    none.grad(grad_q_weight=base, grad_k_weight=base.clone(), accumulate=True)
    assert bool((base == 1).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,heads,kv_heads,dim,rotated", [(1, 32, 8, 128, 128), (200, 8, 2, 128, 128), (37, 5, 1, 80, 40),
                                                          (300, 32, 8, 128, 64), (3, 3, 1, 7, 2)])
def test_gradients_without_an_epsilon(hip_device, monkeypatch, dtype, n, heads, kv_heads, dim, rotated):
    """The formula is finite as long as no head is all zeros: lanes without a head add nothing to the scales' gradients."""
    monkeypatch.setitem(globals(), "EPS", 0.0)
    case = Case(hip_device, dtype, n, heads, kv_heads, dim, rotated)
    case.check(case.run())
    case.check_grads(case.grad())
