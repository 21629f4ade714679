"""The operators of a decoder layer's attention together, as a layer is trained and as it generates, and their calls'
refusals on the device."""
from __future__ import annotations

import ctypes

import pytest
import torch

from slideformer_amd import _lib, _ops_lib, ops

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HIDDEN, HEADS, KV, DIM, EPS = 256, 8, 2, 64, 1e-5
SPLIT = [HEADS * DIM, KV * DIM, KV * DIM]


class Layer:
    def __init__(self, device, seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)

        def normal(std, *shape):
            return (torch.randn(*shape, generator=gen, device=device) * std).to(BF16)

        self.norm, self.q_norm, self.k_norm = ((1 + normal(0.2, n).float()).to(BF16) for n in (HIDDEN, DIM, DIM))
        self.qkv = normal(HIDDEN ** -0.5, sum(SPLIT), HIDDEN)
        self.proj = normal((HEADS * DIM) ** -0.5, HIDDEN, HEADS * DIM)
        angles = torch.arange(512, device=device, dtype=torch.float64)[:, None] * \
            10000.0 ** -(torch.arange(0, DIM, 2, device=device, dtype=torch.float64) / DIM)
        self.cos, self.sin = angles.cos().float(), angles.sin().float()
        self.params = (self.norm, self.qkv, self.q_norm, self.k_norm, self.proj)

    def heads(self, x):
        return [t.unflatten(1, (-1, DIM)) for t in x.split(SPLIT, 1)]

    def forward(self, x, starts, positions):
        h, z, rstd = ops.rms_norm(x, self.norm, eps=EPS)
        qkv = h @ self.qkv.t()
        q, k, v = self.heads(qkv)
        q2, k2 = ops.qk_norm_rotary(q, k, self.cos, self.sin, q_weight=self.q_norm, k_weight=self.k_norm,
                                    positions=positions, eps=EPS)
        out, lse = ops.attention(q2, k2, v, starts=starts)
        return out.flatten(1) @ self.proj.t(), (h, z, rstd, qkv, q2, k2, out, lse)

    def gradients(self, grad, saved, starts, positions):
        """Towards x and the parameters, in self.params' order."""
        h, z, rstd, qkv, q2, k2, out, lse = saved
        q, k, v = self.heads(qkv)
        grad_qkv = torch.empty_like(qkv)                     # written in parts, a view for each
        gq, gk, gv = self.heads(grad_qkv)
        grad_proj = grad.t() @ out.flatten(1)
        grad_out = (grad @ self.proj).unflatten(1, (HEADS, DIM))
        ops.attention_grad(grad_out, q2, k2, v, out, lse, starts=starts, grads=(gq, gk, gv))
        _, _, grad_q_norm, grad_k_norm = ops.qk_norm_rotary_grad(
            gq, gk, q, k, self.cos, self.sin, q_weight=self.q_norm, k_weight=self.k_norm, positions=positions, eps=EPS,
            out=(gq, gk))                                    # over themselves
        grad_h = grad_qkv @ self.qkv
        grad_x, grad_norm = ops.rms_norm_grad(grad_h, z, rstd, self.norm)
        return grad_x, (grad_norm, grad_qkv.t() @ h, grad_q_norm, grad_k_norm, grad_proj)


def _plain(layer, x, params, lengths):
    """The layer in torch, in the parameters' type."""
    norm, w, q_norm, k_norm, proj = params

    def rms(t, scales):
        return t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt() * scales

    def turn(t, n):
        a, b = t[..., :DIM // 2], t[..., DIM // 2:]
        cos, sin = (c[:n, None].to(t.dtype) for c in (layer.cos, layer.sin))
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    outs = []
    for part in x.split(lengths):
        n = len(part)
        q, k, v = layer.heads(rms(part, norm) @ w.t())
        q, k = turn(rms(q, q_norm), n), turn(rms(k, k_norm), n)
        k, v = (t.repeat_interleave(HEADS // KV, 1).transpose(0, 1) for t in (k, v))
        s = q.transpose(0, 1) @ k.transpose(1, 2) * DIM ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -float("inf"))
        outs.append((s.softmax(2) @ v).transpose(0, 1).flatten(1) @ proj.t())
    return torch.cat(outs)


def _inputs(device, lengths):
    gen = torch.Generator(device=device).manual_seed(1)
    x = torch.randn(sum(lengths), HIDDEN, generator=gen, device=device).to(BF16)
    starts = torch.tensor([sum(lengths[:k]) for k in range(len(lengths) + 1)], device=device)
    positions = torch.cat([torch.arange(n, device=device) for n in lengths])
    return gen, x, starts, positions


def test_a_layers_gradients_are_autograds(hip_device):
    """Against float64 autograd on the same bfloat16 parameters.  The longest way through the layer and back rounds
    sixteen times to bfloat16: nine values on the way and seven gradients, of at most 2^-8 each."""
    layer, lengths = Layer(hip_device), [70, 1, 200, 33]
    gen, x, starts, positions = _inputs(hip_device, lengths)
    out, saved = layer.forward(x, starts, positions)
    grad = torch.randn(out.shape, generator=gen, device=hip_device).to(BF16)
    grad_x, grads = layer.gradients(grad, saved, starts, positions)
    leaves = [t.double().requires_grad_() for t in (x, *layer.params)]
    want = _plain(layer, leaves[0], leaves[1:], lengths)
    assert float((out.double() - want.detach()).norm() / want.detach().norm()) < 9 * 2.0 ** -8
    want.backward(grad.double())
    for got, leaf in zip((grad_x, *grads), leaves):
        assert float((got.double() - leaf.grad).norm() / leaf.grad.norm()) < 16 * 2.0 ** -8, tuple(leaf.shape)


def test_a_layer_generates_what_it_would_have_read(hip_device):
    """A prompt and then token after token against a cache gives what the whole text gives at once, within the roundings
    of the way there."""
    layer, lengths = Layer(hip_device, 3), [90, 90]
    _, x, starts, positions = _inputs(hip_device, lengths)
    want, _ = layer.forward(x, starts, positions)
    want = want.view(2, 90, HIDDEN)
    x = x.view(2, 90, HIDDEN)
    cache_k, cache_v = (torch.full((2, 128, KV, DIM), float("nan"), dtype=BF16, device=hip_device) for _ in range(2))

    def step(first, count):
        part = x[:, first:first + count].reshape(-1, HIDDEN)
        at = torch.arange(first, first + count, device=hip_device).repeat(2)
        h, _, _ = ops.rms_norm(part, layer.norm, eps=EPS)
        q, k, v = layer.heads(h @ layer.qkv.t())
        q, k = ops.qk_norm_rotary(q, k, layer.cos, layer.sin, q_weight=layer.q_norm, k_weight=layer.k_norm, positions=at,
                                  eps=EPS)
        cache_k[:, first:first + count] = k.view(2, count, KV, DIM)
        cache_v[:, first:first + count] = v.reshape(2, count, KV, DIM)
        keys = torch.full((2,), first + count, dtype=torch.int32, device=hip_device)
        out, _ = ops.attention(q.view(2, count, HEADS, DIM), cache_k, cache_v, key_lengths=keys)
        return (out.view(2 * count, HEADS * DIM) @ layer.proj.t()).view(2, count, HIDDEN)

    got = [step(0, 40)] + [step(n, 1) for n in range(40, 70)] + [step(70, 20)]
    got = torch.cat(got, 1)
    assert float((got.double() - want.double()).norm() / want.double().norm()) < 4 * 2.0 ** -8


def test_a_key_head_written_into_a_cache_in_place(hip_device):
    """`out` may be rows of a cache, whose other rows stay."""
    gen, q, k = torch.Generator(device=hip_device).manual_seed(2), *(torch.ones(6, h, 64, dtype=BF16, device=hip_device)
                                                                     for h in (4, 2))
    q.normal_(generator=gen), k.normal_(generator=gen)
    table = torch.randn(6, 32, generator=gen, device=hip_device)
    want = ops.qk_norm_rotary(q, k, table, table)
    cache = torch.full((20, 2, 64), 7.0, dtype=BF16, device=hip_device)
    ops.qk_norm_rotary(q, k, table, table, out=(q.clone(), cache[5:11]))
    assert torch.equal(cache[5:11], want[1]) and bool((cache[:5] == 7).all()) and bool((cache[11:] == 7).all())


def test_calls_on_two_streams_at_once(hip_device):
    """Each has workspaces of its own."""
    gen = torch.Generator(device=hip_device).manual_seed(4)
    calls = []
    for n, keys in ((1, 6000), (300, 300)):
        q = torch.randn(2, n, 8, 64, generator=gen, device=hip_device).to(BF16)
        k, v = (torch.randn(2, keys, 2, 64, generator=gen, device=hip_device).to(BF16) for _ in range(2))
        calls.append((q, k, v))
    want = [(r, ops.attention_grad(c[0], *c, *r)) for c in calls for r in [ops.attention(*c)]]
    streams = [torch.cuda.Stream() for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for c, s in zip(calls, streams):
            with torch.cuda.stream(s):
                r = ops.attention(*c)
                got.append((r, ops.attention_grad(c[0], *c, *r)))
    torch.cuda.synchronize()
    for k, (r, g) in enumerate(got):
        for a, b in zip((*r, *g), (*want[k % 2][0], *want[k % 2][1])):
            assert torch.equal(a, b)


@pytest.fixture
def t(hip_device):
    def make(*shape, dtype=BF16):
        return torch.zeros(*shape, dtype=dtype, device=hip_device)
    return make


def test_refusals_of_attention(hip_device, t):
    q, k = t(5, 4, 64), t(5, 2, 64)
    starts, lengths = torch.tensor([0, 5], device=hip_device), torch.tensor([5], device=hip_device)
    lse = t(5, 4, dtype=torch.float32)

    def refused(what, *args, **how):
        with pytest.raises(RuntimeError, match=what):
            ops.attention(*args, **how)

    refused("need starts", q, k, k)
    refused("lengths go with a batch", q, k, k, starts=starts, lengths=lengths)
    refused("starts go with packed", q[None], k[None], k[None], starts=starts)
    refused("cannot share", t(5, 3, 64), k, k, starts=starts)
    refused("size mismatch: v", q, k, t(5, 2, 32), starts=starts)
    refused("size mismatch: k", q, t(5, 2, 32), t(5, 2, 32), starts=starts)
    refused("need key_starts", q, t(6, 2, 64), t(6, 2, 64), starts=starts)
    refused("k is torch.float16", q, k.half(), k.half(), starts=starts)
    refused("unsupported dtype", q.float(), k.float(), k.float(), starts=starts)
    refused("not supported", t(5, 4, 136), t(5, 2, 136), t(5, 2, 136), starts=starts)
    refused("window", q, k, k, starts=starts, window=0)
    refused("window", q, k, k, starts=starts, window=3, causal=False)
    refused("scale", q, k, k, starts=starts, scale=0.0)
    refused("scale", q, k, k, starts=starts, scale=float("nan"))
    refused("unsupported dtype of starts", q, k, k, starts=starts.float())
    refused("key_starts is torch.int32", q, k, k, starts=starts, key_starts=starts.int())
    refused("size mismatch: lengths", q[None], k[None], k[None], lengths=starts)
    refused("need key_lengths", q[None], t(1, 6, 2, 64), t(1, 6, 2, 64), lengths=lengths)
    refused("must be contiguous", t(5, 4, 128)[..., ::2], k, k, starts=starts)
    refused("expected cuda", q, k, k, starts=starts.cpu())
    refused("expected a HIP device", q, k.cpu(), k, starts=starts)
    for what, how in (("grad_out", dict(grad_out=t(5, 4, 32))), ("out is torch.float16", dict(out=q.half())),
                      ("lse", dict(lse=lse[:4])), ("lse is", dict(lse=lse.half())),
                      ("overlap", dict(grads=(t(4, 64).expand(5, 4, 64), k, k.clone()))),
                      ("grad_k", dict(grads=(q.clone(), q.clone(), k.clone())))):
        call = dict(grad_out=q, q=q, k=k, v=k, out=q, lse=lse, starts=starts)
        with pytest.raises(RuntimeError, match=what):
            ops.attention_grad(**{**call, **how})


@pytest.mark.parametrize("packed", [True, False])
def test_gradients_do_not_go_where_the_call_reads(hip_device, t, packed):
    """One kernel would write what the next reads.  Parts of one projection's gradient are fine, and so is
    memory beside what is read."""
    rows = (130,) if packed else (2, 65)
    qkv, new = t(*rows, 8, 64), torch.zeros(*rows, 8, 64, dtype=torch.bfloat16, device=hip_device)
    q, k, v = qkv[..., :4, :], qkv[..., 4:6, :], qkv[..., 6:, :]
    how = dict(starts=torch.tensor([0, 60, 130], device=hip_device)) if packed else {}
    out, lse = ops.attention(q, k, v, **how)
    g = t(*rows, 4, 64)
    want = ops.attention_grad(g, q, k, v, out, lse, **how)
    parts = (new[..., :4, :], new[..., 4:6, :], new[..., 6:, :])
    ops.attention_grad(g, q, k, v, out, lse, grads=parts, **how)
    for a, b in zip(parts, want):
        assert torch.equal(a, b)
    for grads in ((q, k, v), (g, *parts[1:]), (out, *parts[1:]), (parts[0], k, parts[2]), (parts[0], parts[1], v),
                  (parts[0], parts[1], parts[1])):
        kept = [x.clone() for x in grads]
        with pytest.raises(RuntimeError, match="la_attention_grad"):
            ops.attention_grad(g, q, k, v, out, lse, grads=grads, **how)
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    table, w, n = t(130, 32, dtype=torch.float32), t(64), 130
    q, k = q.reshape(n, 4, 64).clone(), k.reshape(n, 2, 64).clone()
    k4 = t(n, 4, 64)
    with pytest.raises(RuntimeError, match="la_qk_norm_rotary"):
        ops.qk_norm_rotary(q, k4, table, table, out=(k4, k4))
    with pytest.raises(RuntimeError, match="la_qk_norm_rotary_grad"):
        ops.qk_norm_rotary_grad(q, k4, q, k4, table, table, out=(q, q))
    with pytest.raises(RuntimeError, match="la_qk_norm_rotary_grad"):
        ops.qk_norm_rotary_grad(q, k, q, k, table, table, q_weight=w, k_weight=w, grad_q_weight=w, grad_k_weight=w)


def test_refusals_of_the_rotation(hip_device, t):
    q, k, table = t(5, 4, 64), t(5, 2, 64), t(5, 32, dtype=torch.float32)

    def refused(what, *args, **how):
        with pytest.raises(RuntimeError, match=what):
            ops.qk_norm_rotary(*args, **how)

    refused("three|3 dimensions", q[None], k, table, table)
    refused("size mismatch: k", q, t(4, 2, 64), table, table)
    refused("k is torch.float16", q, k.half(), table, table)
    refused("not supported", t(5, 1, 258), t(5, 1, 258), table, table)
    refused("cos", q, k, t(5, 33, dtype=torch.float32), t(5, 33, dtype=torch.float32))
    refused("sin", q, k, table, table[:4])
    refused("float32", q, k, table.bfloat16(), table)
    refused("contiguous", q, k, t(5, 64, dtype=torch.float32)[:, ::2], table)
    refused("q_weight", q, k, table, table, q_weight=t(32))
    refused("unsupported dtype of k_weight", q, k, table, table, k_weight=t(64, dtype=torch.float32))
    refused("positions", q, k, table, table, positions=t(4, dtype=torch.int64))
    refused("overlap", q, k, table, table, out=(t(4, 64).expand(5, 4, 64), k))
    refused(r"out\[1\]", q, k, table, table, out=(q, q))
    w = t(64)
    with pytest.raises(RuntimeError, match="accumulate needs"):
        ops.qk_norm_rotary_grad(q, k, q, k, table, table, q_weight=w, accumulate=True)
    with pytest.raises(RuntimeError, match="without its weight"):
        ops.qk_norm_rotary_grad(q, k, q, k, table, table, grad_q_weight=w)
    with pytest.raises(RuntimeError, match="one type"):
        ops.qk_norm_rotary_grad(q, k, q, k, table, table, q_weight=w, k_weight=w, grad_q_weight=t(64),
                                grad_k_weight=t(64, dtype=torch.float32))


@pytest.mark.parametrize("stream", [False, True])
def test_out_of_memory_is_torchs_error(hip_device, t, stream):
    """On the path in Python and on the native one; the next call works."""
    side = torch.cuda.current_stream() if stream else None
    q, k = t(8192, 16, 64), t(8192, 16, 64)
    table, starts = t(8192, 32, dtype=torch.float32), torch.tensor([0, 8192], device=hip_device)
    out, lse = ops.attention(q, k, k, starts=starts)
    calls = (lambda: ops.attention(q, k, k, starts=starts, stream=side),
             lambda: ops.attention_grad(q, q, k, k, out, lse, starts=starts, stream=side),
             lambda: ops.qk_norm_rotary(q, k, table, table, stream=side),
             lambda: ops.qk_norm_rotary_grad(q, k, q, k, table, table, stream=side))
    total = torch.cuda.get_device_properties(hip_device).total_memory
    for call in calls:
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved(hip_device) / total, hip_device)
        held = []                                            # what is free between other tensors
        try:
            while True:
                held.append(torch.empty(1 << 23, dtype=torch.uint8, device=hip_device))
        except torch.OutOfMemoryError:
            pass
        try:
            with pytest.raises(torch.OutOfMemoryError):
                call()
        finally:
            del held
            torch.cuda.set_per_process_memory_fraction(1.0, hip_device)
        call()
        torch.cuda.synchronize()


def _normal(t, *shape, dtype=BF16):
    return t(*shape, dtype=dtype).normal_(generator=torch.Generator(device="cuda").manual_seed(sum(shape)))


def _moved(x, by):
    """The same view `by` elements on in its memory."""
    return x.as_strided(x.shape, x.stride(), x.storage_offset() + by)


def test_rotated_heads_go_to_their_own_place_or_where_nothing_is_read(hip_device, t):
    """Heads are read and written in no order, so a result that lies over others that are read, or over the other result, is
    refused; parts of one projection's rows are fine."""
    n = 130
    wide = _normal(t, n + 2, 16, 64)
    q, k, free, more = (wide[1:-1, 4 * i:4 * i + 4] for i in range(4))
    table, at, scales = _normal(t, n, 32, dtype=torch.float32), t(n * 16, dtype=torch.int64), _normal(t, n * 64)
    at[:n] = torch.arange(n, device=hip_device).flip(0)
    how = dict(q_weight=scales[64:128], k_weight=scales[128:192], positions=at[:n])
    want = ops.qk_norm_rotary(q, k, table, table, **how)
    kept = wide.clone()
    for out in ((k, q), (k, more), (free, q), (_moved(q, 16 * 64), more), (_moved(q, -64), more), (_moved(q, 1), more),
                (free, _moved(k, 64)), (free, _moved(k, -63)), (q, _moved(k, -64)), (free, free), (free, _moved(free, 64)),
                (_moved(free, 16 * 64), free), (free, _moved(free, 3 * 64 + 63))):
        with pytest.raises(RuntimeError, match="la_qk_norm_rotary"):
            ops.qk_norm_rotary(q, k, table, table, out=out, **how)
        assert torch.equal(wide, kept)
    for over in (table, at, scales):                         # heads over the other inputs
        with pytest.raises(RuntimeError, match="la_qk_norm_rotary"):
            ops.qk_norm_rotary(q, k[:, :1], table, table, out=(free, over.view(BF16).view(n, 1, 64)), **how)
    for out in ((free, more), (q, more), (more, k), (q, k)):
        wide.copy_(kept)
        ops.qk_norm_rotary(q, k, table, table, out=out, **how)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        others = torch.ones_like(wide, dtype=torch.bool)
        for x in out:
            others.as_strided(x.shape, x.stride(), x.storage_offset()).zero_()
        assert torch.equal(wide[others], kept[others])


def test_gradients_of_rotated_heads_go_to_their_own_place_or_where_nothing_is_read(hip_device, t):
    n = 130
    wide = _normal(t, n + 2, 24, 64)
    q, k, gq, gk, free, more = (wide[1:-1, 4 * i:4 * i + 4] for i in range(6))
    table, scales = _normal(t, n, 32, dtype=torch.float32), _normal(t, 4, 64)
    normed = dict(q_weight=scales[0], k_weight=scales[1])
    kept = wide.clone()

    def refused(out, how=normed, **more):
        with pytest.raises(RuntimeError, match="la_qk_norm_rotary_grad"):
            ops.qk_norm_rotary_grad(gq, gk, q, k, table, table, out=out, **how, **more)
        assert torch.equal(wide, kept)

    for out in ((gk, gq), (k, q), (gk, more), (free, gq), (free, q), (k, more), (_moved(gq, 64), more), (_moved(q, -64), more),
                (free, _moved(gk, 24 * 64)), (free, _moved(k, 1)), (free, _moved(free, 64)), (free, free)):
        refused(out)
    refused((free, more), grad_q_weight=free[0, 0], grad_k_weight=scales[2])
    refused((free, more), grad_q_weight=scales[2], grad_k_weight=more[n - 1, 3])
    refused((free, more), grad_q_weight=scales.view(-1)[128:192], grad_k_weight=scales.view(-1)[160:224])
    refused((gk, more), how={})
    refused((free, _moved(free, 64)), how={})
    for how, outs in ((normed, ((free, more), (gq, gk), (q, k), (gq, k), (free, gk))),
                      ({}, ((free, more), (gq, gk), (_moved(q, -64), _moved(k, -64)), (k, q)))):      # q and k are not read
        want = ops.qk_norm_rotary_grad(gq, gk, q, k, table, table, **how)
        for out in outs:
            got = ops.qk_norm_rotary_grad(gq, gk, q, k, table, table, out=out, **how)
            for a, b in zip(got, want):
                assert a is b is None or torch.equal(a, b)
            wide.copy_(kept)


def _fp32_within(wide, first):
    """Four fp32 to each row of `wide`, from its element `first` on."""
    return wide.view(torch.float32)[..., 0, :4].as_strided((*wide.shape[:-2], 4), (*(n // 2 for n in wide.stride()[:-2]), 1), first // 2)


@pytest.mark.parametrize("packed", [True, False])
def test_gradients_of_attention_do_not_go_into_one_another(hip_device, t, packed):
    """Nor into lse.  Between all that is read and written is fine, row by row."""
    rows = (130,) if packed else (2, 65)
    wide = _normal(t, *rows, 25, 64)
    q, g, out, gq = (wide[..., 4 * i:4 * i + 4, :] for i in range(4))
    k, v, gk, gv = (wide[..., 16 + 2 * i:18 + 2 * i, :] for i in range(4))
    how = dict(starts=torch.tensor([0, 60, 130], device=hip_device)) if packed else {}
    o, lse = ops.attention(q, k, v, **how)
    out.copy_(o)
    want = ops.attention_grad(g, q, k, v, out, lse, **how)
    kept = wide.clone()

    def refused(grads, lse=lse):
        with pytest.raises(RuntimeError, match="la_attention_grad"):
            ops.attention_grad(g, q, k, v, out, lse, grads=grads, **how)
        assert torch.equal(wide, kept)

    for grads in ((gq, gk, _moved(gk, 64)), (gq, _moved(gv, 64), gv), (gq, _moved(gk, 65), gv), (_moved(gq, 64 * 8 - 63), gk, gv),
                  (_moved(gq, -1), gk, gv), (gq, _moved(gk, -64), gv), (gq, gk, _moved(gk, 1)), (gq, gk, gk), (gq, gv, gv)):
        refused(grads)
    for first in (12 * 64 + 100, 21 * 64 + 56, 22 * 64 - 2):     # the last from grad_k's last element on
        refused((gq, gk, gv), lse=_fp32_within(wide, first))
    within = _fp32_within(wide, 24 * 64 + 8)
    within.copy_(lse)
    kept.copy_(wide)
    for a, b in zip(ops.attention_grad(g, q, k, v, out, within, grads=(gq, gk, gv), **how), want):
        assert torch.equal(a, b)
    for x in (wide, kept):
        for of in (slice(12, 16), slice(20, 24)):
            x[..., of, :] = 0
    assert torch.equal(wide.view(torch.int16), kept.view(torch.int16))       # bits: lse's halves may be NaN


def test_results_of_attention_in_memory_of_the_callers(hip_device, t):
    """Through the C-ABI, which takes out and lse: not where the call reads, indices among it, nor in one another."""
    wide, buf = _normal(t, 4, 14, 64), torch.tensor([0, 3, 4] + [4] * 253, device=hip_device)
    q, k, v, free = wide[:, :4], wide[:, 4:6], wide[:, 6:8], wide[:, 8:12]
    starts, lse = buf[:3], _fp32_within(wide, 13 * 64)
    want = ops.attention(q, k, v, starts=starts)
    lib, kept = _ops_lib.load(), wide.clone()

    def run(out, lse):
        device, call = ops._attention_call(q, k, v, True, None, None, starts, None, None, None)
        call.out, call.lse = ops._heads(out, "out", device, 3), ops._row_values(lse, "lse", device, q)
        work = torch.empty(1 << 16, dtype=torch.uint8, device=device)
        assert lib.la_attention_workspace(ctypes.byref(call)) <= work.numel()
        return lib.la_attention(ctypes.byref(call), work.data_ptr(), work.numel(), torch.cuda.current_stream().cuda_stream)

    for out, where in ((q, lse), (_moved(q, 64), lse), (wide[:, 5:9], lse), (_moved(free, -65), lse), (buf.view(BF16).view(4, 4, 64), lse),
                       (free, _fp32_within(wide, 9 * 64)), (free, _fp32_within(wide, 12 * 64 - 2)), (free, _fp32_within(wide, 6)),
                       (free, _fp32_within(wide, 8 * 64 - 2)), (free, buf.view(torch.float32)[2:18].view(4, 4))):
        assert run(out, where) == _lib.LA_EINVAL
        assert torch.equal(wide, kept) and buf[:4].tolist() == [0, 3, 4, 4]
    assert run(free, lse) == _lib.LA_OK
    assert torch.equal(free, want[0]) and torch.equal(lse, want[1])
    assert torch.equal(wide[:, :8], kept[:, :8])
