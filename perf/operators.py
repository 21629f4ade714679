"""The operators at a language model's two ends, as cases that can be timed.

``embed``       rows of the embedding matrix for a batch of tokens, scaled;
``embed_grad``  the embedding matrix's whole gradient from the grads of those rows;
``norm``        the residual's addition and the root-mean-square norm over it;
``norm_grad``   the gradient of both, towards the sum and the scales;
``norm_8bit``   the norm with its output in 8-bit integers and a scale for each token;
``loss``        softmax cross entropy of hidden states against a vocabulary matrix, a value for each token;
``loss_grad``   its mean, with the gradients of the hidden states and of the matrix.

With ``own`` the framework's operators run, without it elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
IGNORE = -100


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _embed(kind, tokens, vocab, hidden, dtype, scale=1.0):
    return {"kind": kind, "tokens": tokens, "vocab": vocab, "hidden": hidden, "dtype": dtype, "scale": scale}


def _norm(kind, tokens, hidden, dtype):
    return {"kind": kind, "tokens": tokens, "hidden": hidden, "dtype": dtype}


def _loss(kind, tokens, vocab, hidden, dtype, ignored):
    return {"kind": kind, "tokens": tokens, "vocab": vocab, "hidden": hidden, "dtype": dtype, "ignored": ignored}


def listed():
    return [
        # One token's embedding in a Llama-3.1-8B-shaped model: a step of generation, all latency.
        dict(_embed("embed", 1, 128256, 4096, "bf16"), name="embed_one_token"),
        # The embeddings of one training batch of that model.
        dict(_embed("embed", 8192, 128256, 4096, "bf16"), name="embed_batch"),
        # The same batch's gradient of the whole matrix, into the runtime's bf16 grads; frequent tokens repeat.
        dict(_embed("embed_grad", 8192, 128256, 4096, "bf16"), name="embed_grad_batch"),
        # GPT-2 small in fp32, embeddings scaled by the root of the width: short rows, an odd vocabulary.
        dict(_embed("embed_grad", 4095, 50257, 768, "f32", 27.712812921102035), name="embed_grad_gpt2"),
        # The final norm of one generated token.
        dict(_norm("norm", 1, 4096, "bf16"), name="norm_one_token"),
        # A decoder layer's norm over one training batch.
        dict(_norm("norm", 8192, 4096, "bf16"), name="norm_batch"),
        # Its gradient.
        dict(_norm("norm_grad", 8192, 4096, "bf16"), name="norm_grad_batch"),
        # Activations of a 5120-wide layer in 8 bits, an uneven number of tokens.
        dict(_norm("norm_8bit", 1037, 5120, "bf16"), name="norm_8bit_ragged"),
        # The loss of a few held-out tokens: the vocabulary matrix is read once, and that is all the time.
        dict(_loss("loss", 13, 128256, 4096, "bf16", 0.0), name="loss_few_tokens"),
        # A GPT-2-small batch: narrow states, an odd vocabulary, every token trained on.
        dict(_loss("loss_grad", 1024, 50257, 768, "bf16", 0.0), name="loss_grad_gpt2"),
        # A fine-tuning batch of the Llama-3.1-8B shape: a quarter of the tokens are prompt and carry no loss.
        dict(_loss("loss_grad", 4096, 128256, 4096, "bf16", 0.25), name="loss_grad_llama8b"),
        # Nothing fits a tile: odd tokens, odd width, odd vocabulary, fp16, half of the tokens without loss.
        dict(_loss("loss_grad", 515, 32003, 1023, "f16", 0.5), name="loss_grad_odd"),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def _hidden(rng, hi):
    h = _log(rng, 128, hi)
    return h | 1 if rng.random() < 0.25 else max(64, h // 64 * 64)


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "norm", "norm_grad", "norm_8bit", "loss", "loss_grad", "loss_grad"])
    if kind in ("embed", "embed_grad"):
        hidden, vocab = _hidden(rng, 4096), _log(rng, 1000, 128256)
        return _embed(kind, _log(rng, 1, 8192), vocab, hidden, rng.choice(["bf16", "bf16", "f16", "f32"]),
                      rng.choice([1.0, math.sqrt(hidden)]))
    if kind in ("norm", "norm_grad", "norm_8bit"):
        hidden = _hidden(rng, 12288)
        return _norm(kind, _log(rng, 1, max(1, min(16384, 33554432 // hidden))), hidden,
                     rng.choice(["bf16", "bf16", "f16"] + ["f32"] * (kind != "norm_8bit")))
    hidden, vocab = _hidden(rng, 4096), _log(rng, 1000, 128256)
    return _loss(kind, _log(rng, 1, 4096), vocab, hidden, rng.choice(["bf16", "bf16", "f16"]),
                 rng.choice([0.0, 0.25, 0.5]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed * 1009 + 17)
    return gen


def _normal(gen, std, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE).mul_(std)


def _tokens(gen, n, vocab):
    """Token ids in the manner of text: the k-th most frequent token has a share of about 1/k."""
    rank = torch.rand(n, generator=gen, device=DEVICE, dtype=torch.float64).mul_(math.log(vocab)).exp_().long() - 1
    return torch.randperm(vocab, generator=gen, device=DEVICE)[rank.clamp_(0, vocab - 1)]


def prepare(case, seed):
    gen, kind, dtype = _generator(seed), case["kind"], DTYPES[case["dtype"]]
    n, h = case["tokens"], case["hidden"]
    s = {"case": dict(case)}
    if kind in ("embed", "embed_grad"):
        s["tokens"] = _tokens(gen, n, case["vocab"])
        if kind == "embed":
            s["weight"] = _normal(gen, 0.02, case["vocab"], h).to(dtype)
        else:
            s["grad_out"] = _normal(gen, 1e-3, n, h).to(dtype)
            s["grad_weight"] = torch.empty(case["vocab"], h, dtype=dtype, device=DEVICE)
    elif kind in ("norm", "norm_8bit"):
        s["x"] = _normal(gen, 0.5, n, h).to(dtype)
        s["residual"] = _normal(gen, 2.0, n, h).to(dtype)
        s["weight"] = (1 + _normal(gen, 0.2, h)).to(dtype)
    elif kind == "norm_grad":
        s["summed"] = _normal(gen, 2.0, n, h).to(dtype)
        s["rstd"] = (s["summed"].float().square().mean(1) + EPS).rsqrt()
        s["weight"] = (1 + _normal(gen, 0.2, h)).to(dtype)
        s["grad_out"] = _normal(gen, 1e-3, n, h).to(dtype)
        s["grad_summed"] = _normal(gen, 1e-3, n, h).to(dtype)
    else:
        weight = _normal(gen, 0.02, case["vocab"], h)
        targets = _tokens(gen, n, case["vocab"])
        # the states of a model that has learnt something: they lean to their targets, some a lot, some hardly
        lean = torch.rand(n, 1, generator=gen, device=DEVICE) * 8
        s["x"] = (_normal(gen, 1.0, n, h) + lean * (weight[targets] * (50 / math.sqrt(h)))).to(dtype)
        s["weight"] = weight.to(dtype)
        targets[torch.rand(n, generator=gen, device=DEVICE) < case["ignored"]] = IGNORE
        s["targets"] = targets
    return s


# ---------------------------------------------------------------------------
# the plain forms: 32 bits throughout, rounded once at the end
# ---------------------------------------------------------------------------
def _plain_embed(s):
    weight = s["weight"]
    return (weight[s["tokens"]].float() * s["case"]["scale"]).to(weight.dtype)


def _plain_embed_grad(s):
    g = s["grad_out"]
    total = torch.zeros(s["grad_weight"].shape, device=DEVICE)
    total.index_add_(0, s["tokens"], g.float() * s["case"]["scale"])
    return total.to(g.dtype)


def _plain_norm_values(s):
    summed = s["x"].float() + s["residual"].float()
    rstd = (summed.square().mean(1) + EPS).rsqrt()
    return summed, rstd, summed * rstd[:, None] * s["weight"].float()


def _plain_norm(s):
    summed, rstd, out = _plain_norm_values(s)
    return {"out": out.to(s["x"].dtype), "summed": summed.to(s["x"].dtype), "rstd": rstd}


def _plain_norm_8bit(s):
    summed, _, out = _plain_norm_values(s)
    scales = out.abs().amax(1) / 127
    steps = torch.round(out / torch.where(scales > 0, scales, torch.ones_like(scales))[:, None])
    out = (steps.clamp(-127, 127) * scales[:, None]).to(s["x"].dtype)
    return {"out": out, "scales": scales, "summed": summed.to(s["x"].dtype)}


def _plain_norm_grad(s):
    g, weight = s["grad_out"].float(), s["weight"]
    unit = s["summed"].float() * s["rstd"][:, None]
    gw = g * weight.float()
    back = (gw - unit * (gw * unit).mean(1, keepdim=True)) * s["rstd"][:, None] + s["grad_summed"].float()
    return {"grad_x": back.to(weight.dtype), "grad_weight": (g * unit).sum(0).to(weight.dtype)}


def _plain_loss(s, grad):
    x, weight, targets = s["x"], s["weight"], s["targets"]
    xf, wf = x.float(), weight.float()
    keep = targets != IGNORE
    rows = torch.arange(targets.numel(), device=DEVICE)
    at = torch.where(keep, targets, torch.zeros_like(targets))
    p = xf @ wf.t()
    score = p[rows, at]
    top = p.amax(1)
    p.sub_(top[:, None]).exp_()
    total = p.sum(1)
    losses = torch.where(keep, top + total.log() - score, torch.zeros_like(top))
    if not grad:
        return {"loss": losses}
    count = keep.sum().clamp(min=1).float()
    loss = losses.sum() / count
    p.div_(total[:, None])
    p[rows, at] -= 1
    p.mul_((keep.float() / count)[:, None])
    return {"loss": loss, "grad_x": (p @ wf).to(x.dtype), "grad_weight": (p.t() @ xf).to(x.dtype)}


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _own(s):
    from slideformer_amd import ops

    c = s["case"]
    kind = c["kind"]
    if kind == "embed":
        return ops.embedding(s["tokens"], s["weight"], scale=c["scale"])
    if kind == "embed_grad":
        return ops.embedding_grad(s["tokens"], s["grad_out"], s["grad_weight"], scale=c["scale"])
    if kind == "norm":
        out, summed, rstd = ops.rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"])
        return {"out": out, "summed": summed, "rstd": rstd}
    if kind == "norm_8bit":
        steps, scales, summed = ops.rms_norm_8bit(s["x"], s["weight"], eps=EPS, residual=s["residual"])
        out = torch.mul(steps, scales[:, None], out=torch.empty_like(summed))   # the values that the steps stand for
        return {"out": out, "scales": scales, "summed": summed}
    if kind == "norm_grad":
        grad_x, grad_weight = ops.rms_norm_grad(s["grad_out"], s["summed"], s["rstd"], s["weight"],
                                                grad_summed=s["grad_summed"])
        return {"grad_x": grad_x, "grad_weight": grad_weight}
    if kind == "loss":
        return {"loss": ops.linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORE,
                                                 reduction="none")}
    loss, grad_x, grad_weight = ops.linear_cross_entropy_grad(s["x"], s["weight"], s["targets"], ignore_index=IGNORE)
    return {"loss": loss, "grad_x": grad_x, "grad_weight": grad_weight}


_PLAIN = {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "norm": _plain_norm, "norm_8bit": _plain_norm_8bit,
          "norm_grad": _plain_norm_grad, "loss": lambda s: _plain_loss(s, False),
          "loss_grad": lambda s: _plain_loss(s, True)}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, n, h, size = case["kind"], case["tokens"], case["hidden"], SIZES[case["dtype"]]
    if kind == "embed":
        return {"bytes": 8 * n + 2 * n * h * size, "flops": n * h}
    if kind == "embed_grad":
        return {"bytes": 8 * n + (n + case["vocab"]) * h * size, "flops": 2 * n * h}
    if kind == "norm":
        return {"bytes": 4 * n * h * size + h * size + 4 * n, "flops": 5 * n * h}
    if kind == "norm_8bit":
        return {"bytes": n * h * (3 * size + 1) + h * size + 4 * n, "flops": 8 * n * h}
    if kind == "norm_grad":
        return {"bytes": 4 * n * h * size + 2 * h * size + 4 * n, "flops": 10 * n * h}
    v, trained = case["vocab"], n * (1 - case["ignored"])
    if kind == "loss":
        return {"bytes": (trained + v) * h * size + 8 * n + 4, "flops": 2 * trained * v * h}
    # the products of the scores, of the states' gradient and of the matrix's
    return {"bytes": 2 * (n + v) * h * size + 8 * n + 4, "flops": 6 * trained * v * h}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_embed_grad(s, case):
    order = torch.argsort(s["tokens"], stable=True)
    tokens, counts = torch.unique_consecutive(s["tokens"][order], return_counts=True)
    running = torch.zeros(order.numel() + 1, case["hidden"], dtype=torch.float64, device=DEVICE)
    torch.cumsum(s["grad_out"].double()[order], 0, out=running[1:])
    ends = counts.cumsum(0)
    got = torch.zeros(case["vocab"], case["hidden"], dtype=torch.float64, device=DEVICE)
    got[tokens] = (running[ends] - running[ends - counts]) * case["scale"]
    return got


def _exact_norm(s, case):
    h = case["hidden"]
    if case["kind"] == "norm_grad":
        z, g, w, r = (s[k].double() for k in ("summed", "grad_out", "weight", "rstd"))
        inner = torch.mv(g * z, w) / h * r ** 3
        grad = r[:, None] * (g * w) - inner[:, None] * z + s["grad_summed"].double()
        return {"grad_x": grad, "grad_weight": torch.mv((g * z).t().contiguous(), r)}
    z = s["x"].double().add_(s["residual"])
    size = (torch.linalg.vector_norm(z, dim=1).square() / h + EPS).sqrt()
    out = z / size[:, None] * s["weight"].double()
    if case["kind"] == "norm":
        return {"out": out, "summed": z, "rstd": 1 / size}
    scales = torch.linalg.vector_norm(out, ord=math.inf, dim=1) / 127
    # which of two neighbouring steps a value near their middle takes is the rounding's choice: no value of its own
    return {"out": None, "scales": scales, "summed": z}


def _exact_loss(s, case):
    grad = case["kind"] == "loss_grad"
    trained = torch.nonzero(s["targets"] != IGNORE).flatten()
    w = s["weight"].double()
    count = max(1, trained.numel())
    losses = torch.zeros(case["tokens"], dtype=torch.float64, device=DEVICE)
    grad_x = torch.zeros(s["x"].shape, dtype=torch.float64, device=DEVICE) if grad else None
    grad_w = torch.zeros_like(w) if grad else None
    for rows in trained.split(512):
        x, at = s["x"][rows].double(), s["targets"][rows][:, None]
        scores = x @ w.t()
        logp = scores - torch.logsumexp(scores, 1, keepdim=True)
        losses[rows] = -logp.gather(1, at)[:, 0]
        if grad:
            d = logp.exp_().scatter_add_(1, at, torch.full(at.shape, -1.0, dtype=torch.float64, device=DEVICE))
            d /= count
            grad_x[rows] = d @ w
            grad_w.addmm_(d.t(), x)
    return {"loss": losses.sum() / count, "grad_x": grad_x, "grad_weight": grad_w} if grad else {"loss": losses}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        return s["weight"].double()[s["tokens"]] * case["scale"]
    if case["kind"] == "embed_grad":
        return _exact_embed_grad(s, case)
    if case["kind"] in ("loss", "loss_grad"):
        return _exact_loss(s, case)
    return _exact_norm(s, case)
