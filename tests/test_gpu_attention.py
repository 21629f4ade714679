"""Attention and its gradient against plain 64-bit computations.

Tolerances are bounds on the operators' own roundings, element by element.  ``U`` is one
rounding to the operands' type, ``U32`` one to fp32.  A score is an fp32 sum of dim products,
off by at most dim * U32 times the sum of their sizes; with the multiplication by scale * log2(e), the
difference from the row's maximum or lse and the exponential's own error a probability is off by
E = that + (|score| + |lse| + 2) * 4 * U32, relative.  It is rounded to 16 bits once before it is
multiplied, and sums of n terms in fp32 are off by n * U32 times the sum of their sizes.  float16 has fewer
exponents: what lies below 2^-14 of a row's largest probability is off by up to 2^-25 of it.
"""
from __future__ import annotations

import pytest
import torch

from slideformer_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25}              # half the smallest number
FLOOR = {BF16: 0.0, F16: 2.0 ** -25}
U32 = 2.0 ** -24
NAN = float("nan")


def _normal(gen, std, *shape):
    return torch.randn(*shape, generator=gen, device=gen.device).mul_(std)


def _within(got, want, bound, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    off[(got == want)] = 0                               # infinities
    bad = ~(off <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(off[bad].max()),
                                 float((off / bound.clamp(min=1e-300)).max()))


class Case:
    """Sequences of given lengths, packed or as a padded batch, with all that the operators take."""

    def __init__(self, device, dtype, queries, keys, heads, kv_heads, dim, packed=True, causal=True, window=None, scale=None,
                 index=torch.int32, rows=None, key_rows=None, before=0, behind=0, lay=None, seed=0):
        gen = torch.Generator(device=device).manual_seed(seed + 7 * dim + heads)
        self.dtype, self.queries, self.keys, self.heads, self.kv, self.dim = dtype, queries, keys, heads, kv_heads, dim
        self.packed, self.causal, self.window = packed, causal, window
        self.scale = dim ** -0.5 if scale is None else scale
        self.where = {}
        lay = lay or (lambda t: t)
        if packed:
            n, m = (before + sum(x) + behind for x in (queries, keys))
            self.at = [slice(before + sum(queries[:b]), before + sum(queries[:b + 1])) for b in range(len(queries))]
            self.key_at = [slice(before + sum(keys[:b]), before + sum(keys[:b + 1])) for b in range(len(keys))]
            self.where["starts"] = torch.tensor([s.start for s in self.at] + [self.at[-1].stop], dtype=index, device=device)
            if queries != keys:
                self.where["key_starts"] = torch.tensor([s.start for s in self.key_at] + [self.key_at[-1].stop], dtype=index,
                                                        device=device)
            shape, key_shape = (n,), (m,)
        else:
            rows, key_rows = rows or max(queries), key_rows or max(keys)
            self.at = [(b, slice(0, n)) for b, n in enumerate(queries)]
            self.key_at = [(b, slice(0, m)) for b, m in enumerate(keys)]
            shape, key_shape = (len(queries), rows), (len(keys), key_rows)
            if any(n != rows for n in queries):
                self.where["lengths"] = torch.tensor(queries, dtype=index, device=device)
            if "lengths" in self.where or any(m != key_rows for m in keys):
                self.where["key_lengths"] = torch.tensor(keys, dtype=index, device=device)
        q = _normal(gen, 2.0, *shape, heads, dim).to(dtype)
        k = _normal(gen, 1.0, *key_shape, kv_heads, dim).to(dtype)
        v = _normal(gen, 1.0, *key_shape, kv_heads, dim).to(dtype)
        g = _normal(gen, 1.0, *shape, heads, dim).to(dtype)
        # what no sequence has is never looked at
        self.mine, self.my_keys = (torch.zeros(s, dtype=torch.bool, device=device) for s in (shape, key_shape))
        for at, key_at in zip(self.at, self.key_at):
            self.mine[at] = True
            self.my_keys[key_at] = True
        for t in (q, g):
            t[~self.mine] = NAN
        for t in (k, v):
            t[~self.my_keys] = NAN
        self.q, self.k, self.v, self.g = (lay(t) for t in (q, k, v, g))
        self.how = dict(causal=causal, window=window, scale=scale, **self.where)

    def run(self, **more):
        return ops.attention(self.q, self.k, self.v, **self.how, **more)

    def grad(self, out, lse, **more):
        return ops.attention_grad(self.g, self.q, self.k, self.v, out, lse, **self.how, **more)

    def pieces(self):
        """For every sequence: rows' places, keys' places, which keys each query sees, and q, k, v, g by head in fp64."""
        for at, key_at, n, m in zip(self.at, self.key_at, self.queries, self.keys):
            last = torch.arange(n, device=self.q.device)[:, None] + (m - n)
            key = torch.arange(m, device=self.q.device)
            sees = key <= last if self.causal else torch.ones(n, m, dtype=torch.bool, device=self.q.device)
            if self.window:
                sees = sees & (key > last - self.window)
            group = self.heads // self.kv
            q, g = (t[at].double().transpose(0, 1) for t in (self.q, self.g))
            k, v = (t[key_at].double().transpose(0, 1).repeat_interleave(group, 0) for t in (self.k, self.v))
            yield at, key_at, sees, q, k, v, g

    def check(self, out, lse):
        u, tiny = U[self.dtype], TINY[self.dtype]
        assert bool((out[~self.mine] == 0).all()) and bool((lse[~self.mine] == -float("inf")).all())
        for at, _, sees, q, k, v, _ in self.pieces():
            s = (q @ k.transpose(1, 2) * self.scale).masked_fill(~sees, -float("inf"))
            want_lse = torch.logsumexp(s, 2) if s.shape[2] else torch.full(s.shape[:2], -float("inf"), device=s.device)
            p = (s - want_lse.nan_to_num(neginf=0.0)[..., None]).exp()
            want = p @ v
            n = s.shape[2]
            off = (self.dim * U32 * self.scale * (q.abs() @ k.abs().transpose(1, 2))).masked_fill(~sees, 0)
            e = off + (s.masked_fill(~sees, 0).abs() + want_lse.nan_to_num(neginf=0.0).abs()[..., None] + 2) * 4 * U32
            worst = e.amax(2, keepdim=True) if n else torch.zeros(*s.shape[:2], 1, device=s.device)
            # the probability's own rounding, its error and that of the sum that it is divided by, both sums
            bound = u * want.abs() + ((u + 2 * worst + 2 * (n + 8) * U32) * p.abs() + FLOOR[self.dtype] * sees) @ v.abs() + tiny
            _within(out[at].transpose(0, 1), want, bound, "out")
            _within(lse[at].transpose(0, 1), want_lse,
                    worst[..., 0] + (n + 8) * U32 + want_lse.nan_to_num(neginf=0.0).abs() * 4 * U32, "lse")

    def check_grads(self, grads, out, lse, exact=False):
        """The formula with the out and lse that were given."""
        u, tiny = U[self.dtype], TINY[self.dtype]
        gq, gk, gv = grads
        assert bool((gq[~self.mine] == 0).all())
        assert bool((gk[~self.my_keys] == 0).all()) and bool((gv[~self.my_keys] == 0).all())
        group = self.heads // self.kv
        for at, key_at, sees, q, k, v, g in self.pieces():
            n, m = sees.shape
            s = (q @ k.transpose(1, 2) * self.scale).masked_fill(~sees, -float("inf"))
            row_lse = lse[at].double().transpose(0, 1).nan_to_num(neginf=0.0)
            p = (s - row_lse[..., None]).exp()
            off = self.dim * U32 * self.scale * (q.abs() @ k.abs().transpose(1, 2))
            e = off + (s.masked_fill(~sees, 0).abs() + row_lse.abs()[..., None] + 2) * 4 * U32
            o = out[at].double().transpose(0, 1)
            dp, delta = g @ v.transpose(1, 2), (g * o).sum(2, keepdim=True)
            # delta from out, or from P and dP where a row sees few keys: what lies between is out's rounding
            own = (p * dp).sum(2, keepdim=True)
            if exact:
                delta, gap = own, (4 * e.amax(2, keepdim=True) if m else 0) * (p * dp.abs()).sum(2, keepdim=True) + \
                    2 * (m + 8) * U32 * (p * dp.abs()).sum(2, keepdim=True)
            else:
                gap = (own - delta).abs() * (1 + 2.0 ** -12) + 2.0 ** -12 * own.abs()
            ds = p * (dp - delta)
            dp_off = self.dim * U32 * (g.abs() @ v.abs().transpose(1, 2) + (g.abs() * o.abs()).sum(2, keepdim=True)) + gap
            ds_off = ds.abs() * (u + e + 4 * U32) + p * (dp_off + 2 * U32 * (dp.abs() + delta.abs()))
            if self.dtype == F16 and ds.numel():
                # held within a wave times a power of two that brings the largest to 2^10 at least
                ds_off = ds_off + ds.abs().amax((1, 2), keepdim=True) * 2.0 ** -35 * sees
            dq, dk, dv = ds @ k * self.scale, ds.transpose(1, 2) @ q * self.scale, p.transpose(1, 2) @ g
            dq_off = (ds_off + m * U32 * ds.abs()) @ k.abs() * self.scale
            dk_off = (ds_off + n * group * U32 * ds.abs()).transpose(1, 2) @ q.abs() * self.scale
            dv_off = ((u + e + n * group * U32) * p + FLOOR[self.dtype] * 2.0 ** -14 * sees).transpose(1, 2) @ g.abs()
            dk, dv, dk_off, dv_off = (t.unflatten(0, (self.kv, group)).sum(1) for t in (dk, dv, dk_off, dv_off))
            for got, want, bound, name in ((gq[at], dq, dq_off, "grad_q"), (gk[key_at], dk, dk_off, "grad_k"),
                                           (gv[key_at], dv, dv_off, "grad_v")):
                _within(got.transpose(0, 1), want, (u + 4 * U32) * want.abs() + (1 + u) * bound + tiny, name)

    def all(self):
        out, lse = self.run()
        self.check(out, lse)
        grads = self.grad(out, lse)
        self.check_grads(grads, out, lse)
        # a fixed order: equal bits
        again = self.run()
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
        for a, b in zip(self.grad(out, lse), grads):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (4, 2, 128), (6, 2, 80), (8, 1, 32), (3, 3, 63), (5, 5, 8),
                                                (7, 1, 128), (2, 1, 100)])
@pytest.mark.parametrize("lengths", [[1], [2], [33], [64], [65], [130], [300], [1, 0, 77, 128, 3], [0, 0, 5, 0]])
def test_packed_sequences(hip_device, dtype, heads, kv_heads, dim, lengths):
    Case(hip_device, dtype, lengths, lengths, heads, kv_heads, dim).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal,window", [(False, None), (True, 1), (True, 2), (True, 50), (True, 64), (True, 1000)])
@pytest.mark.parametrize("dim", [64, 128])
def test_masks(hip_device, dtype, causal, window, dim):
    Case(hip_device, dtype, [1, 63, 200, 400, 129], [1, 63, 200, 400, 129], 4, 2, dim, causal=causal, window=window).all()


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (BF16, 72)])
@pytest.mark.parametrize("queries,keys", [([5, 70, 200], [100, 30, 150]), ([1, 1, 1], [1, 0, 700]), ([140, 0, 3], [0, 50, 3]),
                                          ([128, 256], [64, 1])])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 40), (False, None)])
def test_queries_and_keys_of_different_lengths(hip_device, dtype, dim, queries, keys, causal, window):
    """Among them rows that see nothing: causal ones before the keys begin, and sequences without keys."""
    Case(hip_device, dtype, queries, keys, 4, 2, dim, causal=causal, window=window).all()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF16, 4, 2, 64), (F16, 8, 1, 128)])
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (True, 30)])
@pytest.mark.parametrize("queries,keys", [([5, 200, 64, 0], [100, 30, 0, 9]), ([700, 3], [2, 200])])
def test_padded_keys_have_no_gradient(hip_device, dtype, heads, kv_heads, dim, causal, window, queries, keys):
    """Whole tiles of them, and some beside a sequence's own keys."""
    Case(hip_device, dtype, queries, keys, heads, kv_heads, dim, packed=False, causal=causal, window=window,
         rows=max(queries) + 20, key_rows=300).all()


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF16, 2, 1, 64), (F16, 24, 8, 100), (BF16, 5, 5, 128)])
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (True, 40)])
@pytest.mark.parametrize("queries,keys,rows", [([1], [1300], 6), ([3, 1, 0, 2], [90, 300, 70, 1], 8), ([20], [200], 100)])
def test_padded_queries_see_nothing(hip_device, dtype, heads, kv_heads, dim, causal, window, queries, keys, rows):
    """Beside whole tiles of keys that the sequence's own queries see."""
    Case(hip_device, dtype, queries, keys, heads, kv_heads, dim, packed=False, causal=causal, window=window, rows=rows,
         key_rows=max(keys) + 30).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64), (3, 3, 128), (8, 1, 96)])
@pytest.mark.parametrize("lengths,how", [([2], {}), ([3, 2, 6, 1], {}), ([60, 5], dict(causal=False)), ([500, 131], dict(window=2)),
                                         ([400], dict(window=5)), ([300], dict(window=33))])
def test_gradients_of_rows_that_see_few_keys(hip_device, dtype, heads, kv_heads, dim, lengths, how):
    """dP - delta is small there beside both, and out's rounding is not: delta is that of P and dP."""
    case = Case(hip_device, dtype, lengths, lengths, heads, kv_heads, dim, **how)
    out, lse = case.run()
    case.check_grads(case.grad(out, lse), out, lse, exact=True)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("keys", [10, 64, 300])
def test_gradients_of_a_share_of_the_keys(hip_device, dtype, keys):
    """With out and lse over all keys, calls over pieces of them give these pieces' gradients, and add up."""
    case = Case(hip_device, dtype, [40], [2 * keys], 4, 2, 64, packed=False, causal=False)
    out, lse = case.run()
    gq, gk, gv = case.grad(out, lse)
    halves = [ops.attention_grad(case.g, case.q, case.k[:, s].contiguous(), case.v[:, s].contiguous(), out, lse, causal=False)
              for s in (slice(0, keys), slice(keys, 2 * keys))]
    for whole, at in ((gk, 1), (gv, 2), (gq, 0)):
        got = halves[0][0].double() + halves[1][0].double() if at == 0 else torch.cat([h[at] for h in halves], 1).double()
        # delta is out's in the halves and may be its own in the whole: each element within out's rounding
        assert float((got - whole.double()).norm() / whole.double().norm()) < 8 * U[dtype]


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("packed", [True, False])
def test_rows_of_no_sequence(hip_device, index, packed):
    """Zeros in new tensors, as they were in given ones; what they hold (here NaN) reaches nothing."""
    lengths = [50, 1, 100]
    case = Case(hip_device, BF16, lengths, lengths, 4, 2, 64, packed=packed, index=index, before=5, behind=140, rows=170,
                key_rows=170)
    case.all()
    out, lse = case.run()
    want = case.grad(out, lse)
    given = tuple(torch.full_like(t, 3.0) for t in (case.q, case.k, case.v))
    got = case.grad(out, lse, grads=given)
    for g, w, mine in zip(got, want, (case.mine, case.my_keys, case.my_keys)):
        assert torch.equal(g[mine], w[mine]) and bool((g[~mine] == 3).all())
    assert all(a is b for a, b in zip(got, given))


def test_a_row_that_sees_one_key_has_its_value_and_no_gradient(hip_device):
    for dtype in (BF16, F16):
        for how in (dict(lengths=[1] * 50), dict(lengths=[90], window=1)):
            lengths = how.pop("lengths")
            case = Case(hip_device, dtype, lengths, lengths, 6, 3, 128, **how)
            out, lse = case.run()
            assert torch.equal(out, case.v.repeat_interleave(2, 1))
            gq, gk, gv = case.grad(out, lse)
            assert bool((gq == 0).all()) and bool((gk == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("keys,capacity", [([1, 2, 31], 40), ([32, 33, 64, 127, 0], 128), ([5000, 1, 2049], 5000),
                                           ([9001], 9001), ([700] * 20, 701)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (9, 1, 96), (40, 1, 128), (64, 2, 64)])
def test_one_new_token_against_a_cache(hip_device, dtype, keys, capacity, heads, kv_heads, dim):
    """Keys are shared out among workgroups where there are few sequences, and among waves."""
    case = Case(hip_device, dtype, [1] * len(keys), keys, heads, kv_heads, dim, packed=False, key_rows=capacity)
    out, lse = case.run()
    if 0 in keys:                                        # causal, but without a key
        assert bool((out[keys.index(0)] == 0).all())
    case.check(out, lse)
    again = case.run()
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("queries,keys", [(3, 4100), (16, 900), (77, 77), (100, 6000), (300, 3500)])
@pytest.mark.parametrize("window", [None, 600])
def test_a_piece_of_a_prompt_against_a_cache(hip_device, queries, keys, window):
    case = Case(hip_device, BF16, [queries, queries], [keys, keys - 13], 4, 2, 128, packed=False, window=window)
    case.all()


def test_long_sequences(hip_device):
    Case(hip_device, BF16, [2500], [2500], 2, 1, 128).all()
    Case(hip_device, F16, [1900, 2300], [1900, 2300], 2, 1, 64, packed=False).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("how", [dict(), dict(window=500), dict(causal=False), dict(packed=False, rows=1200, key_rows=1200)])
def test_gradients_of_few_keys_with_many_rows(hip_device, dtype, how):
    """Several workgroups share the rows that see a key, and add their sums at the end."""
    lengths = [1100, 0, 40, 260]
    case = Case(hip_device, dtype, lengths, lengths, 8, 1, 128, before=3, behind=150, **how)
    case.all()
    out, lse = case.run()
    want = case.grad(out, lse)
    given = tuple(torch.full_like(t, 3.0) for t in (case.q, case.k, case.v))
    for g, w, mine in zip(case.grad(out, lse, grads=given), want, (case.mine, case.my_keys, case.my_keys)):
        assert torch.equal(g[mine], w[mine]) and bool((g[~mine] == 3).all())
    few = Case(hip_device, dtype, [1500], [70], 8, 1, 128, causal=False)
    few.all()


def _fused(t):
    """Heads as they lie in the rows of a wider matrix."""
    wide = torch.full((*t.shape[:-2], t.shape[-2] + 3, t.shape[-1]), NAN, dtype=t.dtype, device=t.device)
    wide[..., 1:-2, :] = t
    return wide[..., 1:-2, :]


def _heads_first(t):
    return t.transpose(-3, -2).contiguous().transpose(-3, -2)


def _odd(t):
    """One element into its memory, rows an odd number of elements apart."""
    size = (*t.shape[:-2], t.shape[-2] * t.shape[-1] + 1)
    buf = torch.full((t.new_empty(size, device="meta").numel() + 1,), NAN, dtype=t.dtype, device=t.device)
    view = buf[1:].view(size)[..., :-1].unflatten(-1, t.shape[-2:])
    view.copy_(t)
    return view


@pytest.mark.parametrize("lay", [_fused, _heads_first, _odd])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_views_of_any_order(hip_device, lay, packed, dim):
    lengths = [150, 33]
    case = Case(hip_device, BF16, lengths, lengths, 4, 2, dim, packed=packed, lay=lay)
    case.all()
    plain = Case(hip_device, BF16, lengths, lengths, 4, 2, dim, packed=packed)
    out, lse = case.run()
    want, want_lse = plain.run()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    given = tuple(lay(torch.zeros_like(t)) for t in (plain.q, plain.k, plain.v))
    order = torch.empty(lse.shape[::-1], device=hip_device).permute(*reversed(range(lse.dim())))    # heads first
    case.grad(lay(out), order.copy_(lse), grads=given)
    for got, w, mine in zip(given, plain.grad(out, lse), (case.mine, case.my_keys, case.my_keys)):
        assert torch.equal(got[mine], w[mine])


def test_distances_that_pass_32_bits(hip_device):
    """2600 rows, 2 MiB apart: 5 GiB."""
    rows, step = 2600, 1 << 20
    buf = torch.empty(rows * step, dtype=BF16, device=hip_device)
    case = Case(hip_device, BF16, [1], [rows], 8, 2, 128, packed=False)
    want, want_lse = case.run()
    far = buf.as_strided((1, rows, 2, 128), (0, step, 128, 1))
    far.copy_(case.k)
    case.k = far
    out, lse = case.run()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    # a row so far from the next that a tile's rows are out of a descriptor's reach: copied first
    few = buf.as_strided((1, 70, 2, 128), (0, 35 << 20, 128, 1))
    case = Case(hip_device, BF16, [70], [70], 4, 2, 128, packed=False)
    want, want_lse = case.run()
    few.copy_(case.v)
    case.v = few
    out, lse = case.run()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_large_and_bad_scores(hip_device):
    """Scores in the thousands, rows of equal scores, and what infinities and NaN in a sequence give: NaN rows."""
    case = Case(hip_device, BF16, [200], [200], 2, 1, 64, scale=40.0)
    case.check(*case.run())
    case = Case(hip_device, BF16, [200], [200], 2, 1, 64)
    case.k[:] = 1.0
    case.check(*case.run())
    # a key that is NaN: rows that see it are NaN, rows that do not are as before
    want, want_lse = case.run()
    case.k[150] = NAN
    out, lse = case.run()
    assert bool(out[150:].isnan().all()) and bool(lse[150:].isnan().all())
    assert torch.equal(out[:150], want[:150]) and torch.equal(lse[:150], want_lse[:150])


def test_gradients_far_from_one_in_fp16(hip_device):
    """Grads scaled by powers of two come out scaled: as long as the results have a normal number for it."""
    case = Case(hip_device, F16, [300], [300], 4, 2, 128)
    out, lse = case.run()
    want = case.grad(out, lse)
    for power in (-6, 5, 9):
        scaled = ops.attention_grad((case.g.float() * 2.0 ** power).half(), case.q, case.k, case.v, out, lse, **case.how)
        for a, b in zip(scaled, want):
            a, b = a.float(), b.float() * 2.0 ** power
            normal = b.abs() >= 2.0 ** -12
            assert bool(((a - b).abs()[normal] <= b.abs()[normal] * 2.0 ** -10 + 2.0 ** (power - 20)).all())


def test_gradients_are_difference_quotients(hip_device):
    """Of sum(c * out) along a direction, by the 64-bit formula on the operator's own inputs."""
    case = Case(hip_device, BF16, [90, 40], [90, 40], 4, 2, 64)
    out, lse = case.run()
    grads = case.grad(out, lse)
    gen = torch.Generator(device=hip_device).manual_seed(5)

    def loss(q, k, v):
        total = 0.0
        for (at, key_at, sees, *_, g) in case.pieces():
            qd, kd, vd = q[at].transpose(0, 1), *(t[key_at].transpose(0, 1).repeat_interleave(2, 0) for t in (k, v))
            p = (qd @ kd.transpose(1, 2) * case.scale).masked_fill(~sees, -float("inf")).softmax(2)
            total = total + (p @ vd * g).sum()
        return float(total)

    base = [t.double() for t in (case.q, case.k, case.v)]
    for i, grad in enumerate(grads):
        direction = torch.randn(grad.shape, generator=gen, device=hip_device, dtype=torch.float64)
        h = 1e-5
        ahead, back = ([t + sign * h * direction if j == i else t for j, t in enumerate(base)] for sign in (1, -1))
        slope = (loss(*ahead) - loss(*back)) / (2 * h)
        # each element is within about three roundings to bfloat16 of its size; signs are independent of the direction's
        bound = 3 * U[BF16] * float(grad.double().norm()) * 4
        assert abs(float((grad.double() * direction).sum()) - slope) < bound


@pytest.mark.parametrize("form", ["packed", "step"])
def test_captured_and_replayed(hip_device, form):
    if form == "packed":
        case = Case(hip_device, BF16, [100, 70], [100, 70], 4, 2, 128)
    else:
        case = Case(hip_device, BF16, [1, 1], [4000, 3000], 8, 2, 128, packed=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = case.run()
        case.grad(out, lse)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = case.run()
        grads = case.grad(out, lse)
    for step in range(4):
        gen = torch.Generator(device=hip_device).manual_seed(100 + step)
        for t in (case.q, case.k, case.v, case.g):
            t.copy_(torch.randn(t.shape, generator=gen, device=hip_device))
        graph.replay()
        want, want_lse = case.run()                      # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        for a, b in zip(grads, case.grad(want, want_lse)):
            assert torch.equal(a, b)


def test_on_another_stream(hip_device):
    case = Case(hip_device, BF16, [700, 20], [700, 20], 4, 2, 128)
    want, want_lse = case.run()
    want_grads = case.grad(want, want_lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, lse = case.run(stream=side)
    grads = case.grad(out, lse, stream=side)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    for a, b in zip(grads, want_grads):
        assert torch.equal(a, b)


def test_windows_longer_than_any_sequence(hip_device):
    case = Case(hip_device, BF16, [70], [70], 2, 1, 64)
    want = case.run()
    for window in (70, 1 << 32, 1 << 40, (1 << 64) + 1):
        for side in (None, torch.cuda.current_stream()):
            got = ops.attention(case.q, case.k, case.v, window=window, starts=case.where["starts"], stream=side)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_nothing_to_do(hip_device):
    empty = torch.empty(0, 4, 64, dtype=BF16, device=hip_device)
    keys = torch.ones(0, 2, 64, dtype=BF16, device=hip_device)
    starts = torch.zeros(3, dtype=torch.int32, device=hip_device)
    out, lse = ops.attention(empty, keys, keys, starts=starts)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    assert [t.shape[0] for t in ops.attention_grad(out, empty, keys, keys, out, lse, starts=starts)] == [0, 0, 0]
    # queries without any key, and keys without any query
    q = torch.ones(2, 3, 4, 64, dtype=BF16, device=hip_device)
    k = torch.ones(2, 0, 2, 64, dtype=BF16, device=hip_device)
    out, lse = ops.attention(q, k, k)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())
    assert bool((ops.attention_grad(q, q, k, k, out, lse)[0] == 0).all())
    none = q[:, :0]
    out, lse = ops.attention(none, q[:, :, :2], q[:, :, :2])
    _, gk, gv = ops.attention_grad(none, none, q[:, :, :2], q[:, :, :2], out, lse)
    assert bool((gk == 0).all()) and bool((gv == 0).all())
    with pytest.raises(RuntimeError, match="starts must have"):
        ops.attention(empty, keys, keys, starts=starts[:1])


def test_indices_beyond_the_rows_stay_within_them(hip_device):
    """They are the caller's mistake; no access leaves the tensors for it."""
    q = torch.ones(100, 4, 64, dtype=BF16, device=hip_device)
    k = torch.ones(100, 2, 64, dtype=BF16, device=hip_device)
    starts = torch.tensor([-5, 60, 1 << 40], device=hip_device)
    good = torch.tensor([0, 60, 100], device=hip_device)
    out, lse = ops.attention(q, k, k, starts=starts)
    want, want_lse = ops.attention(q, k, k, starts=good)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    out, lse = ops.attention(q[None], k[None], k[None], key_lengths=torch.tensor([1 << 35], device=hip_device))
    want, want_lse = ops.attention(q[None], k[None], k[None])
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_many_sequences(hip_device):
    """More than the 64 that are looked through at a time."""
    lengths = [(7 * b) % 23 for b in range(200)]
    Case(hip_device, BF16, lengths, lengths, 2, 1, 64).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (3, 3, 64), (4, 2, 80)])
@pytest.mark.parametrize("window", [2, 3, 8, 32, 64])
@pytest.mark.parametrize("more", [1, 5, 30, 62])
@pytest.mark.parametrize("packed", [True, False])
def test_gradients_of_rows_that_see_few_keys_wherever_these_begin(hip_device, dtype, heads, kv_heads, dim, window, more, packed):
    """With more keys than queries 128 rows' windows begin anywhere in a tile of keys, and reach into four of them."""
    queries = [300, 140]
    case = Case(hip_device, dtype, queries, [n + more for n in queries], heads, kv_heads, dim, packed=packed, window=window)
    out, lse = case.run()
    case.check_grads(case.grad(out, lse), out, lse, exact=True)
