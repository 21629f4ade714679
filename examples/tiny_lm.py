"""A small language model trained with this package alone around its blocks' products.

Embedding, norms and loss are ``slideformer_amd.ops``, every parameter is stepped by
``LayerAdam``, and only the blocks' two matrix products are torch's.  The model is
held as the sliding-window runtime holds one: each layer's fp32 master, its bf16
compute copy and its bf16 grads are flat buffers, the gradients are written into
the flat grads layer by layer, last layer first, and each layer is then stepped
with one global clip.  The vocabulary matrix is tied: the loss writes its gradient,
and the embedding adds its own to it.

    python examples/tiny_lm.py [--steps N]
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from slideformer_amd import LayerAdam, ops

VOCAB, HIDDEN, FFN, BLOCKS, BATCH, LENGTH, EPS = 1000, 192, 512, 3, 8, 64, 1e-5


class Layer:
    """A layer's flat fp32 master, bf16 compute copy and bf16 grads, with views of its parameters."""

    def __init__(self, adam, index, shapes, device, gen):
        sizes = [torch.Size(s).numel() for s in shapes]
        self.adam, self.index = adam, index
        self.master = torch.cat([torch.ones(n, device=device) if len(s) == 1 else
                                 torch.randn(n, generator=gen, device=device) * s[-1] ** -0.5
                                 for s, n in zip(shapes, sizes)])
        self.compute = self.master.bfloat16()
        self.grad = torch.zeros_like(self.compute)
        self.params = [v.view(s) for v, s in zip(self.compute.split(sizes), shapes)]
        self.grads = [v.view(s) for v, s in zip(self.grad.split(sizes), shapes)]
        adam.add_layer_params(index, [torch.nn.Parameter(self.master, requires_grad=False)])

    def step(self, coef):
        group = self.adam.begin_chunk_step(self.index)
        self.adam.step_chunk(self.master, self.grad, self.adam.exp_avg_flat[self.index],
                             self.adam.exp_avg_sq_flat[self.index], group, bf16_out=self.compute, clip_coef=coef)
        self.adam.end_chunk_step(self.index)


class TinyLM:
    def __init__(self, device, seed=0, lr=3e-3):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.adam = LayerAdam(lr=lr, betas=(0.9, 0.95), weight_decay=0.01)
        self.vocab = Layer(self.adam, 0, [(VOCAB, HIDDEN)], device, gen)
        self.blocks = [Layer(self.adam, k + 1, [(HIDDEN,), (FFN, HIDDEN), (HIDDEN, FFN)], device, gen)
                       for k in range(BLOCKS)]
        self.final = Layer(self.adam, BLOCKS + 1, [(HIDDEN,)], device, gen)
        self.device = device

    def forward(self, tokens):
        """The final norm's output for int64 tokens [n], and what backward needs of each layer."""
        saved = []
        x, z = ops.embedding(tokens, self.vocab.params[0]), None
        for block in self.blocks:
            scales, up, down = block.params
            out, z, rstd = ops.rms_norm(x, scales, eps=EPS, residual=z)
            leaves = [t.detach().requires_grad_() for t in (out, up, down)]
            x = torch.nn.functional.silu(leaves[0] @ leaves[1].t()) @ leaves[2].t()
            saved.append((z, rstd, leaves, x))
            x = x.detach()
        out, z, rstd = ops.rms_norm(x, self.final.params[0], eps=EPS, residual=z)
        return out, (z, rstd), saved

    def gradients(self, tokens, targets):
        """Fills every layer's grads, last layer first; returns the loss."""
        out, (z, rstd), saved = self.forward(tokens)
        loss, grad, _ = ops.linear_cross_entropy_grad(out, self.vocab.params[0], targets,
                                                      grad_weight=self.vocab.grads[0])
        # the gradient of the residual stream, which every block's branch adds to
        grad, _ = ops.rms_norm_grad(grad, z, rstd, self.final.params[0], grad_weight=self.final.grads[0])
        for block, (z, rstd, leaves, y) in zip(reversed(self.blocks), reversed(saved)):
            grad_out, grad_up, grad_down = torch.autograd.grad(y, leaves, grad)
            block.grads[1].copy_(grad_up)
            block.grads[2].copy_(grad_down)
            grad, _ = ops.rms_norm_grad(grad_out, z, rstd, block.params[0], grad_summed=grad,
                                        grad_weight=block.grads[0])
        ops.embedding_grad(tokens, grad, self.vocab.grads[0], accumulate=True)
        return loss

    def step(self, tokens, targets, max_norm=1.0):
        loss = self.gradients(tokens, targets)
        layers = [self.final, *reversed(self.blocks), self.vocab]
        norm = self.adam.grad_norm_begin(self.device)
        for layer in layers:
            norm.add(layer.grad)
        coef, _ = norm.finish(max_norm)
        for layer in layers:
            layer.step(coef)
        return loss

    def loss(self, tokens, targets):
        """Mean loss without gradients."""
        return ops.linear_cross_entropy(self.forward(tokens)[0], self.vocab.params[0], targets)


def batches(device, seed=1):
    """Endless synthetic text: each token mostly decides the next; the first tokens of a sequence are prompt."""
    gen = torch.Generator(device=device).manual_seed(seed)
    follows = torch.randint(VOCAB, (VOCAB,), generator=gen, device=device)
    while True:
        rows = [torch.randint(VOCAB, (BATCH,), generator=gen, device=device)]
        for _ in range(LENGTH):
            stray = torch.rand(BATCH, generator=gen, device=device) < 0.1
            other = torch.randint(VOCAB, (BATCH,), generator=gen, device=device)
            rows.append(torch.where(stray, other, follows[rows[-1]]))
        text = torch.stack(rows, 1)
        targets = text[:, 1:].clone()
        targets[:, :LENGTH // 4] = -100
        yield text[:, :-1].reshape(-1), targets.reshape(-1)


def main(steps=150):
    device = torch.device("cuda", 0)
    model, data = TinyLM(device), batches(device)
    held_out = next(batches(device, seed=1))
    first = float(model.loss(*held_out))
    for k in range(steps):
        loss = model.step(*next(data))
        if k % 50 == 0:
            print(f"step {k}: loss {float(loss):.3f}", flush=True)
    last = float(model.loss(*held_out))
    print(f"loss of a batch {first:.3f} -> {last:.3f}", flush=True)
    return first, last


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=150)
    main(parser.parse_args().steps)
