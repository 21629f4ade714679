"""The operators and the optimizer together, as the example trains with them: its
gradients against autograd's through the same model written in torch, and its loss."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("tiny_lm", os.path.join(REPO, "examples", "tiny_lm.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_gradients_are_autograds(example, hip_device):
    """Against float32 autograd on the same bf16 parameters.  The example rounds every activation and gradient
    between operators to bf16, at most 2^-8 relative each, about twenty of them on the longest way."""
    model = example.TinyLM(hip_device)
    tokens, targets = next(example.batches(hip_device))
    loss = model.gradients(tokens, targets)
    layers = [model.vocab, *model.blocks, model.final]
    params = [[p.detach().float().requires_grad_() for p in layer.params] for layer in layers]

    def norm(z, scales):
        return z * (z.square().mean(1, keepdim=True) + example.EPS).rsqrt() * scales

    z = params[0][0][tokens]
    for scales, up, down in params[1:-1]:
        z = z + torch.nn.functional.silu(norm(z, scales) @ up.t()) @ down.t()
    scores = norm(z, params[-1][0]) @ params[0][0].t()
    want = torch.nn.functional.cross_entropy(scores, targets)
    want.backward()
    want = want.detach()
    assert abs(float(loss) - float(want)) < 0.02 * float(want)
    for layer, mine in zip(layers, params):
        for got, p in zip(layer.grads, mine):
            off = (got.float() - p.grad).norm() / p.grad.norm()
            assert float(off) < 20 * 2.0 ** -8, (tuple(p.shape), float(off))


def test_the_example_learns(example, hip_device):
    first, last = example.main(steps=120)
    assert last < 0.7 * first, (first, last)
