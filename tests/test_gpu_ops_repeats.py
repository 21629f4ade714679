"""The embedding's gradient where tokens repeat: few tokens, which are not sorted, and
more, which are, against 64-bit sums; and the time that repeats take."""
from __future__ import annotations

import pytest
import torch

from slideformer_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -149}


def _tokens(kind, n, vocab, device):
    at = torch.arange(n, device=device)
    if kind == "same":
        return torch.full((n,), vocab - 1, device=device)
    if kind == "half":
        return torch.where(at % 2 == 0, torch.zeros_like(at), at % vocab)
    return at * 7 // 16 % vocab                              # runs of two and three, each in one place or two


@pytest.mark.parametrize("kind", ["same", "half", "runs"])
@pytest.mark.parametrize("n", [2, 15, 16, 17, 64, 65, 129, 255, 256, 257])
@pytest.mark.parametrize("dtype,out_dtype,hidden", [(BF16, BF16, 1023), (F16, F32, 513), (F32, F32, 260)])
def test_repeated_tokens(hip_device, kind, n, dtype, out_dtype, hidden):
    vocab, scale = 50, 1.5
    tokens = _tokens(kind, n, vocab, hip_device)
    gen = torch.Generator(device=hip_device).manual_seed(n + hidden)
    grad = torch.randn(n, hidden, generator=gen, device=hip_device).to(dtype)
    got = ops.embedding_grad(tokens, grad, torch.full((vocab, hidden), float("nan"), dtype=out_dtype,
                                                      device=hip_device), scale=scale)
    want = torch.zeros(vocab, hidden, dtype=torch.float64, device=hip_device)
    sizes = torch.zeros_like(want)
    want.index_add_(0, tokens, grad.double() * scale)
    sizes.index_add_(0, tokens, grad.double().abs() * scale)
    count = torch.bincount(tokens, minlength=vocab)[:, None]
    # a sum's chain is no longer than its terms, then the scale's product and the rounding
    bound = U[out_dtype] * want.abs() + (count + 2) * 2.0 ** -24 * sizes + TINY[out_dtype]
    assert not bool(((got.double() - want).abs() > bound).any()) and not bool(got.isnan().any())
    assert bool((got[(count == 0).flatten()] == 0).all())
    # a padding token's rows reach nothing, and its row is cleared
    padding = int(tokens[0])
    grad[tokens == padding] = float("nan")
    padded = ops.embedding_grad(tokens, grad, torch.full_like(got, float("nan")), scale=scale, padding_idx=padding)
    want[padding], bound[padding] = 0, 0
    assert not bool(((padded.double() - want).abs() > bound).any()) and not bool(padded.isnan().any())


def _us(call):
    for _ in range(3):
        call()
    times = []
    for _ in range(7):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(10):
            call()
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end) * 100)
    return sorted(times)[3]


def test_a_repeated_token_does_not_wait_for_one_wave(hip_device):
    """256 equal tokens 4096 wide, the most that are not sorted, against 257, which are.  By one wave, one row after
    the other, they would take twenty times as long."""
    grad = torch.randn(257, 4096, device=hip_device).to(BF16)
    tokens = torch.full((257,), 3, device=hip_device)
    weight = torch.empty(8, 4096, dtype=BF16, device=hip_device)
    few = _us(lambda: ops.embedding_grad(tokens[:256], grad[:256], weight))
    assert few < 3 * _us(lambda: ops.embedding_grad(tokens, grad, weight))
