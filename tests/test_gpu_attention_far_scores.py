"""Attention in float16 of rows whose scores lie far apart, against plain 64-bit computations.

Where one key's score is far above the others', as that of a text's first token often is, most of a row's probabilities
are below what float16 holds beside 1.  They are many, and where that key's value is small the result is theirs.

Tolerances are those of attention's other tests but for the probabilities' floor.  float16 holds them times 2^9 relative
to a reference R that follows the tiles of keys, 64 or 32 of them: half of its smallest step, 2^-25, is 2^-34 R, and R is
at most 2^14 times the sum of a tile's probabilities, or else less than 2^-40 of the row's.  So one is off by at most
2^-20 of its tile's sum; the other term, 2^-74 of the row's, is less than float32's roundings of the row's sum.
"""
from __future__ import annotations

import pytest
import torch

from slideformer_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25}
FLOOR = {BF16: 0.0, F16: 2.0 ** -20}
U32 = 2.0 ** -24


def _scored(device, dtype, batch, rows, heads, kv_heads, dim, levels, value_of_high=0.0):
    """q, k, v whose scores are about `levels` [keys], a little apart; values of the highest keys are `value_of_high`,
    those of the others about 1."""
    gen = torch.Generator(device=device).manual_seed(dim + rows)
    keys = len(levels)

    def normal(std, *shape):
        return torch.randn(*shape, generator=gen, device=device).mul_(std)

    q, k = normal(0.3, batch, rows, heads, dim), normal(0.3, batch, keys, kv_heads, dim)
    v = 1 + normal(0.5, batch, keys, kv_heads, dim)
    high = levels >= levels.max() - 1
    v[:, high] = value_of_high
    q[..., 0] = 8.0
    k[..., 0] = (levels * dim ** 0.5 / 8.0)[:, None]
    return (t.to(dtype) for t in (q, k, v))


def _check(q, k, v, causal):
    """The first and the last sequence's first and last head against the formula, up to some 150 rows of each."""
    out, lse = ops.attention(q, k, v, causal=causal)
    dtype, (batch, rows, heads, dim), (keys, kv) = q.dtype, q.shape, k.shape[1:3]
    u, tiny, floor, scale = U[dtype], TINY[dtype], FLOOR[dtype], dim ** -0.5
    at = torch.arange(0, rows, -(-rows // 150), device=q.device)
    sees = torch.arange(keys, device=q.device) <= (at[:, None] + keys - rows if causal else keys)
    for b, h in {(b, h) for b in (0, batch - 1) for h in (0, heads - 1)}:
        qh, kh, vh = q[b, at, h].double(), *(t[b, :, h // (heads // kv)].double() for t in (k, v))
        s = (qh @ kh.t() * scale).masked_fill(~sees, -float("inf"))
        want_lse = torch.logsumexp(s, 1)
        p = (s - want_lse[:, None]).exp()
        want = p @ vh
        tiles = torch.nn.functional.pad(p, (0, -keys % 64)).unflatten(1, (-1, 64)).sum(2).repeat_interleave(64, 1)[:, :keys]
        e = dim * U32 * scale * (qh.abs() @ kh.abs().t()) + (s.masked_fill(~sees, 0).abs() + want_lse.abs()[:, None] + 2) * 4 * U32
        worst = e.masked_fill(~sees, 0).amax(1, keepdim=True)
        bound = u * want.abs() + ((u + 2 * worst + 2 * (keys + 8) * U32) * p + floor * tiles * sees) @ vh.abs() + tiny
        off = (out[b, at, h].double() - want).abs()
        assert bool((off <= bound).all()), (b, h, float((off / bound).max()), float((off / want.abs().clamp(min=tiny)).max()))
        off = (lse[b, at, h].double() - want_lse).abs()
        bound = worst[:, 0] + (keys + 8) * U32 + want_lse.abs() * 4 * U32
        assert bool((off <= bound).all()), (b, h, "lse", float((off / bound).max()))


# (sequences, rows, query heads, key heads, dim): one token's heads, a few rows, and many; keys shared out among
# workgroups, and, with 512 workgroups without that, each row's gone over by one
FORMS = [(1, 1, 4, 2, 128), (1, 1, 2, 2, 64), (1, 5, 4, 1, 80), (1, 150, 2, 1, 128), (1, 150, 1, 1, 64), (128, 1, 8, 4, 64),
         (1, 2200, 32, 32, 64), (1, 2200, 32, 32, 128)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("above", [9.0, 13.0, 17.5, 22.0, 26.0, 40.0, 200.0])
@pytest.mark.parametrize("at", [0, 700, -1])
def test_one_key_far_above_the_others(hip_device, dtype, form, above, at):
    """Its value is 0, so the result is the others'."""
    levels = torch.zeros(8192, device=hip_device)
    levels[at] = above
    _check(*_scored(hip_device, dtype, *form, levels), causal=1 < form[1] and at == 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("value", [0.0, 1e-3, 5.0])
def test_many_keys_far_below_one(hip_device, form, value):
    levels = torch.zeros(40000 if form[0] == 1 else 5000, device=hip_device)
    levels[3] = 17.5
    _check(*_scored(hip_device, F16, *form, levels, value), causal=False)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("step", [-30.0, -9.0, -3.0, -0.5, 0.5, 3.0, 9.0, 30.0])
def test_scores_that_rise_or_fall_from_tile_to_tile(hip_device, dtype, form, step):
    levels = (torch.arange(1280, device=hip_device) // 64).float() * step
    _check(*_scored(hip_device, dtype, *form, levels, 1.0), causal=False)
    _check(*_scored(hip_device, dtype, *form, levels[:1111], 1.0), causal=1 < form[1] <= 1111)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("apart", [7.0, 12.0, 20.0, 60.0])
@pytest.mark.parametrize("every", [32, 64, 65, 200])
def test_scores_that_go_up_and_down(hip_device, form, apart, every):
    """Rows' references follow them both ways; the upper ones' values are 0."""
    levels = (torch.arange(3000, device=hip_device) // every % 2).float() * apart
    _check(*_scored(hip_device, F16, *form, levels), causal=False)
    levels[levels > 0] += torch.linspace(0, 3, int((levels > 0).sum()), device=hip_device)
    _check(*_scored(hip_device, F16, *form, levels), causal=1 < form[1])
