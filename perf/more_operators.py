"""The operators of a decoder layer's attention, as cases that can be timed.

``rotary``          the root-mean-square norm of every query and key head, and the position rotation after it;
``rotary_grad``     their gradient, towards the heads and the norms' scales;
``attention``       softmax attention of queries over the keys of their sequence, with the rows' log-sum-exp;
``attention_grad``  its gradient, towards queries, keys and values.

With ``own`` the framework's operators run, without it elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
BASE = 500000.0


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _rotary(kind, tokens, heads, kv_heads, dim, rotated, dtype, interleaved=False, norm=True):
    return {"kind": kind, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotated": rotated,
            "dtype": dtype, "interleaved": interleaved, "norm": norm}


def _packed(kind, tokens, sequences, heads, kv_heads, dim, dtype, causal=True, window=0):
    """Sequences of different lengths, one after the other; queries and keys are the same tokens."""
    return {"kind": kind, "layout": "packed", "tokens": tokens, "sequences": sequences, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal, "window": window}


def _batch(kind, sequences, tokens, keys, ragged, heads, kv_heads, dim, dtype, causal=True, window=0):
    """The last ``tokens`` tokens of each sequence against a cache for ``keys`` of them; a ragged one is not full."""
    return {"kind": kind, "layout": "batch", "tokens": tokens, "sequences": sequences, "keys": keys, "ragged": ragged,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal, "window": window}


def listed():
    return [
        # The new token of a step of generation, heads of a Llama-3.1-8B-shaped layer with normed queries and keys: latency.
        dict(_rotary("rotary", 1, 32, 8, 128, 128, "bf16"), name="rotary_one_token"),
        # The same over one training batch.
        dict(_rotary("rotary", 8192, 32, 8, 128, 128, "bf16"), name="rotary_batch"),
        # Its gradient.
        dict(_rotary("rotary_grad", 8192, 32, 8, 128, 128, "bf16"), name="rotary_grad_batch"),
        # Nothing is even: odd tokens, heads of 80 of which 40 turn, in neighbouring pairs, fp16.
        dict(_rotary("rotary_grad", 1037, 16, 2, 80, 40, "f16", True), name="rotary_grad_ragged"),
        # One prompt of a chat, all launch and latency.
        dict(_batch("attention", 1, 77, 77, False, 32, 8, 128, "bf16"), name="attention_prompt"),
        # A step of generation for a batch of chats, caches filled to different lengths.
        dict(_batch("attention", 16, 1, 8192, True, 32, 8, 128, "bf16"), name="attention_step"),
        # A step of generation at the end of one long document.
        dict(_batch("attention", 1, 1, 65536, False, 32, 8, 128, "bf16"), name="attention_long_step"),
        # One training sequence of the Llama-3.1-8B shape.
        dict(_packed("attention", 8192, 1, 32, 8, 128, "bf16"), name="attention_long"),
        # A GPT-2-small batch: short sequences, heads of 64, no shared ones.
        dict(_batch("attention", 8, 1024, 1024, False, 12, 12, 64, "bf16"), name="attention_gpt2"),
        # Its gradient.
        dict(_batch("attention_grad", 8, 1024, 1024, False, 12, 12, 64, "bf16"), name="attention_grad_gpt2"),
        # The gradient of a packed fine-tuning batch of the Llama-3.1-8B shape, five documents of different lengths.
        dict(_packed("attention_grad", 8192, 5, 32, 8, 128, "bf16"), name="attention_grad_packed"),
        # Short odd sequences with a sliding window, heads of 80, fp16.
        dict(_packed("attention_grad", 1501, 7, 10, 5, 80, "f16", True, 200), name="attention_grad_odd"),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def _heads(rng, most):
    kv = _log(rng, 1, 12)
    return max(1, min(most // kv, rng.choice([1, 2, 3, 4, 7, 8]))) * kv, kv


def _dim(rng):
    return rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 2 * rng.randrange(12, 64)])


def draw(rng):
    kind = rng.choice(["rotary", "rotary_grad", "attention", "attention", "attention_grad", "attention_grad"])
    heads, kv = _heads(rng, 32)
    dim = _dim(rng)
    if kind in ("rotary", "rotary_grad"):
        rotated = dim if rng.random() < 0.6 else max(2, dim // rng.choice([2, 4]) // 2 * 2)
        most = max(1, min(8192, 8192 * 40 * 128 // ((heads + kv) * dim)))
        return _rotary(kind, _log(rng, 1, most), heads, kv, dim, rotated, rng.choice(["bf16", "bf16", "f16", "f32"]),
                       rng.random() < 0.3, rng.random() < 0.75)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    window = _log(rng, 1, 1024) if rng.random() < 0.25 else 0
    causal = window > 0 or rng.random() < 0.8
    # how many pairs of a query and a key the largest listed case has time for
    pairs = int(5e11 / ((4 if kind == "attention" else 10) * heads * dim))
    if kind == "attention" and rng.random() < 0.5:
        keys = _log(rng, 1, 32768)
        sequences = _log(rng, 1, max(1, min(32, (1 << 19) // keys)))
        tokens = 1 if rng.random() < 0.6 else _log(rng, 1, min(keys, 100, max(1, pairs // (keys * sequences))))
        return _batch(kind, sequences, tokens, keys, rng.random() < 0.5, heads, kv, dim, dtype, causal, window)
    tokens = _log(rng, 1, min(4096, math.isqrt(pairs)))
    if rng.random() < 0.5:
        sequences = _log(rng, 1, max(1, min(16, 8192 // tokens, pairs // tokens ** 2)))
        return _batch(kind, sequences, tokens, tokens, rng.random() < 0.5, heads, kv, dim, dtype, causal, window)
    return _packed(kind, tokens, _log(rng, 1, max(1, min(16, tokens))), heads, kv, dim, dtype, causal, window)


def _lengths(case):
    """How many tokens each sequence's queries have, and its keys."""
    b = case["sequences"]
    if case["layout"] == "packed":
        # unequal shares of the tokens, the k-th in proportion to 1 / (k + 1)
        shares = [1 / (k + 1) for k in range(b)]
        ends = [round(sum(shares[:k + 1]) / sum(shares) * case["tokens"]) for k in range(b)]
        got = [hi - lo for lo, hi in zip([0, *ends], ends)]
        return got, got
    keys = [case["keys"] - (k * 7919 % max(1, case["keys"] * 3 // 4) if case["ragged"] else 0) for k in range(b)]
    return [min(case["tokens"], k) for k in keys], keys


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed * 1013 + 29)
    return gen


def _normal(gen, std, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE).mul_(std)


def _prepare_rotary(case, gen):
    n, dim, dtype = case["tokens"], case["dim"], DTYPES[case["dtype"]]
    s = {}
    # queries and keys lie in the rows of one projection's output, as do their gradients
    width = (case["heads"] + 2 * case["kv_heads"]) * dim
    rows = _normal(gen, 1.5, n, width).to(dtype)
    split = [case["heads"] * dim, case["kv_heads"] * dim, case["kv_heads"] * dim]
    q, k, _ = rows.split(split, 1)
    s["q"], s["k"] = q.unflatten(1, (-1, dim)), k.unflatten(1, (-1, dim))
    for name in ("q_weight", "k_weight"):
        s[name] = (1 + _normal(gen, 0.2, dim)).to(dtype) if case["norm"] else None
    # the table of a context of 16384 positions; the batch's documents begin at 0, or further on in a long one
    at = torch.arange(16384, device=DEVICE, dtype=torch.float64)
    speed = BASE ** -(torch.arange(0, case["rotated"], 2, device=DEVICE, dtype=torch.float64) / case["rotated"])
    angles = at[:, None] * speed
    s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
    first = torch.randint(0, 16384 - n + 1, (1,), generator=gen, device=DEVICE)
    s["positions"] = first + torch.arange(n, device=DEVICE)
    if case["kind"] == "rotary_grad":
        s["grad_q"] = _normal(gen, 1e-3, n, case["heads"], dim).to(dtype)
        s["grad_k"] = _normal(gen, 1e-3, n, case["kv_heads"], dim).to(dtype)
    return s


def prepare(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    if case["kind"] in ("rotary", "rotary_grad"):
        return {"case": dict(case), **_prepare_rotary(case, gen)}
    s = {"case": dict(case)}
    tokens, keys = _lengths(case)
    if case["layout"] == "packed":
        shape = key_shape = (case["tokens"],)
        starts = [sum(tokens[:k]) for k in range(case["sequences"] + 1)]
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
    else:
        shape, key_shape = (case["sequences"], case["tokens"]), (case["sequences"], case["keys"])
        s["lengths"] = torch.tensor(tokens, dtype=torch.int32, device=DEVICE) if case["ragged"] else None
        s["key_lengths"] = torch.tensor(keys, dtype=torch.int32, device=DEVICE) if case["ragged"] else None
    # queries that look for something: scores spread over a few units
    s["q"] = _normal(gen, 2.0, *shape, case["heads"], case["dim"]).to(dtype)
    s["k"] = _normal(gen, 1.0, *key_shape, case["kv_heads"], case["dim"]).to(dtype)
    s["v"] = _normal(gen, 1.0, *key_shape, case["kv_heads"], case["dim"]).to(dtype)
    if case["kind"] == "attention_grad":
        s["grad_out"] = _normal(gen, 1e-2, *shape, case["heads"], case["dim"]).to(dtype)
        forward = _plain_attention(s)
        s["out"], s["lse"] = forward["out"], forward["lse"]
    return s


# ---------------------------------------------------------------------------
# the plain forms: 32 bits throughout, rounded once at the end
# ---------------------------------------------------------------------------
def _turn(x, cos, sin, rotated, interleaved):
    """The first ``rotated`` elements of every head, in pairs, by the angles of their token."""
    head, rest = x[..., :rotated], x[..., rotated:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :rotated // 2], head[..., rotated // 2:]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([head, rest], -1)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]

    def one(x, weight):
        y = x.float()
        if weight is not None:
            y = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight.float()
        return _turn(y, cos, sin, c["rotated"], c["interleaved"]).to(x.dtype)

    return {"q": one(s["q"], s["q_weight"]), "k": one(s["k"], s["k_weight"])}


def _plain_rotary_grad(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]

    def one(grad, x, weight):
        g = _turn(grad.float(), cos, -sin, c["rotated"], c["interleaved"])
        if weight is None:
            return g.to(grad.dtype), None
        y = x.float()
        rstd = (y.square().mean(-1, keepdim=True) + EPS).rsqrt()
        unit, gw = y * rstd, g * weight.float()
        back = (gw - unit * (gw * unit).mean(-1, keepdim=True)) * rstd
        return back.to(grad.dtype), (g * unit).sum((0, 1)).to(weight.dtype)

    grad_q, q_weight = one(s["grad_q"], s["q"], s["q_weight"])
    grad_k, k_weight = one(s["grad_k"], s["k"], s["k_weight"])
    return {"grad_q": grad_q, "grad_k": grad_k, "grad_q_weight": q_weight, "grad_k_weight": k_weight}


def _padded(s):
    """Which row of the flat tensors every place of a padded batch holds, (queries, keys), and the lengths of both."""
    c = s["case"]
    if c["layout"] == "packed":
        starts = s["starts"].long()
        lengths = starts[1:] - starts[:-1]
        at = starts[:-1, None] + torch.arange(max(_lengths(c)[0]), device=DEVICE)
        at = at.clamp_(max=c["tokens"] - 1)
        return at, at, lengths, lengths
    b = c["sequences"]
    lengths = torch.full((b,), c["tokens"], device=DEVICE) if s["lengths"] is None else s["lengths"].long()
    key_lengths = torch.full((b,), c["keys"], device=DEVICE) if s["key_lengths"] is None else s["key_lengths"].long()
    at = torch.arange(b * c["tokens"], device=DEVICE).view(b, -1)
    return at, torch.arange(b * c["keys"], device=DEVICE).view(b, -1), lengths, key_lengths


def _by_head(x, at, kv_heads):
    """Rows of x [.., heads, dim] as fp32 [batch, kv_heads, group of heads * length, dim]."""
    x = x.flatten(0, -3)[at].float()
    b, n, heads, dim = x.shape
    return x.view(b, n, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, dim)


def _by_token(x, s, length, heads):
    """The inverse, for values [batch, kv_heads, group * length, ..] of the queries' or the keys' places."""
    c = s["case"]
    b, kv = x.shape[:2]
    x = x.view(b, kv, heads // kv, length, -1).permute(0, 3, 1, 2, 4).reshape(b, length, heads, -1)
    if c["layout"] == "packed":
        token = torch.arange(c["tokens"], device=DEVICE)
        sequence = torch.searchsorted(s["starts"].long(), token, right=True) - 1
        x = x[sequence, token - s["starts"].long()[sequence]]
    return x


def _plain_scores(s):
    """Heads in fp32, scores with the masked ones at -inf, and the padded sizes."""
    c = s["case"]
    kv = c["kv_heads"]
    at, key_at, lengths, key_lengths = _padded(s)
    q, k, v = _by_head(s["q"], at, kv), _by_head(s["k"], key_at, kv), _by_head(s["v"], key_at, kv)
    n, m = at.shape[1], key_at.shape[1]
    row, key = torch.arange(n, device=DEVICE)[:, None], torch.arange(m, device=DEVICE)
    seen = (row < lengths[:, None, None]) & (key < key_lengths[:, None, None])
    last = row + (key_lengths - lengths)[:, None, None]      # the last key that a causal row sees
    if c["causal"]:
        seen = seen & (key <= last)
    if c["window"]:
        seen = seen & (key > last - c["window"])
    scores = q @ k.transpose(-1, -2)
    scores.mul_(c["dim"] ** -0.5)
    scores.view(len(lengths), kv, -1, n, m).masked_fill_(~seen[:, None, None], -math.inf)
    return q, k, v, scores, n, m


def _plain_softmax(scores):
    """In place; returns the log-sum-exp. Rows that see nothing: zeros, and -inf."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    total = scores.sub_(top).exp_().sum(-1, keepdim=True)
    scores.div_(torch.where(total > 0, total, 1.0))
    return top + total.log()


def _plain_attention(s):
    c = s["case"]
    _, _, v, p, n, _ = _plain_scores(s)
    lse = _plain_softmax(p)
    out = _by_token(p @ v, s, n, c["heads"]).to(s["q"].dtype)
    return {"out": out, "lse": _by_token(lse, s, n, c["heads"]).squeeze(-1)}


def _plain_attention_grad(s):
    c = s["case"]
    q, k, v, p, n, m = _plain_scores(s)
    _plain_softmax(p)
    at, _, lengths, _ = _padded(s)
    grad = s["grad_out"].flatten(0, -3)[at] * (torch.arange(n, device=DEVICE) < lengths[:, None])[..., None, None]
    grad = _by_head(grad, torch.arange(at.numel(), device=DEVICE).view(at.shape), c["kv_heads"])
    grad_v = p.transpose(-1, -2) @ grad
    d = grad @ v.transpose(-1, -2)
    d.sub_((d * p).sum(-1, keepdim=True)).mul_(p).mul_(c["dim"] ** -0.5)
    grads = (d @ k, d.transpose(-1, -2) @ q, grad_v)
    sizes = ((n, c["heads"]), (m, c["kv_heads"]), (m, c["kv_heads"]))
    return {name: _by_token(x, s, *size).to(s["q"].dtype)
            for name, x, size in zip(("grad_q", "grad_k", "grad_v"), grads, sizes)}


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _own(s):
    from slideformer_amd import ops

    c = s["case"]
    kind = c["kind"]
    if kind == "rotary":
        q, k = ops.qk_norm_rotary(s["q"], s["k"], s["cos"], s["sin"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                                  positions=s["positions"], eps=EPS, interleaved=c["interleaved"])
        return {"q": q, "k": k}
    if kind == "rotary_grad":
        grad_q, grad_k, q_weight, k_weight = ops.qk_norm_rotary_grad(
            s["grad_q"], s["grad_k"], s["q"], s["k"], s["cos"], s["sin"], q_weight=s["q_weight"],
            k_weight=s["k_weight"], positions=s["positions"], eps=EPS, interleaved=c["interleaved"])
        return {"grad_q": grad_q, "grad_k": grad_k, "grad_q_weight": q_weight, "grad_k_weight": k_weight}
    where = {"starts": s["starts"]} if c["layout"] == "packed" else {"lengths": s["lengths"],
                                                                     "key_lengths": s["key_lengths"]}
    window = c["window"] or None
    if kind == "attention":
        out, lse = ops.attention(s["q"], s["k"], s["v"], causal=c["causal"], window=window, **where)
        return {"out": out, "lse": lse}
    grad_q, grad_k, grad_v = ops.attention_grad(s["grad_out"], s["q"], s["k"], s["v"], s["out"], s["lse"],
                                                causal=c["causal"], window=window, **where)
    return {"grad_q": grad_q, "grad_k": grad_k, "grad_v": grad_v}


_PLAIN = {"rotary": _plain_rotary, "rotary_grad": _plain_rotary_grad, "attention": _plain_attention,
          "attention_grad": _plain_attention_grad}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _pairs(case):
    """How many keys the queries of one head see, all told."""
    total = 0
    for n, m in zip(*_lengths(case)):
        if not case["causal"]:
            total += n * m
            continue
        window = case["window"] or m
        total += sum(max(0, min(window, m - n + i + 1)) for i in range(n))
    return total


def work(case):
    size, heads, kv, dim = SIZES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] in ("rotary", "rotary_grad"):
        n = case["tokens"]
        values = n * (heads + kv) * dim
        extra = 8 * n + 4 * n * case["rotated"]              # positions, and a row of both tables
        if case["kind"] == "rotary":
            return {"bytes": 2 * values * size + extra, "flops": (4 + 4 * case["norm"]) * values}
        return {"bytes": (2 + case["norm"]) * values * size + extra, "flops": (4 + 12 * case["norm"]) * values}
    queries, keys = (sum(x) for x in _lengths(case))
    pairs = _pairs(case)
    rows = queries * heads
    if case["kind"] == "attention":
        return {"bytes": (2 * rows + 2 * keys * kv) * dim * size + 4 * rows, "flops": 4 * dim * pairs * heads}
    # the queries, out and their gradients; keys, values and theirs; five products
    return {"bytes": (4 * rows + 4 * keys * kv) * dim * size + 4 * rows, "flops": 10 * dim * pairs * heads}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_rotary(s, case):
    """Norm and rotation of one head's row as a linear map's parts: pairs as complex numbers, turned by a product."""
    r = case["rotated"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]

    def turned(x, turn):
        head = x[..., :r]
        pairs = torch.complex(head[..., 0::2], head[..., 1::2]) if case["interleaved"] else \
            torch.complex(head[..., :r // 2], head[..., r // 2:])
        pairs = pairs * turn
        head = torch.view_as_real(pairs).flatten(-2) if case["interleaved"] else torch.cat([pairs.real, pairs.imag], -1)
        return torch.cat([head, x[..., r:]], -1)

    if case["kind"] == "rotary":
        got = {}
        for name in ("q", "k"):
            x = s[name].double()
            if case["norm"]:
                x = x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True).square() / case["dim"] + EPS).sqrt()
                x = x * s[name + "_weight"].double()
            got[name] = turned(x, turn)
        return got
    got = {"grad_q": None, "grad_k": None, "grad_q_weight": None, "grad_k_weight": None}
    for name in ("q", "k"):
        g = turned(s["grad_" + name].double(), turn.conj())
        if case["norm"]:
            x = s[name].double()
            size = (torch.linalg.vector_norm(x, dim=-1, keepdim=True).square() / case["dim"] + EPS).sqrt()
            got["grad_" + name + "_weight"] = (g * x / size).flatten(0, 1).sum(0)
            g = g * s[name + "_weight"].double()
            g = g / size - x * ((g * x).sum(-1, keepdim=True) / (case["dim"] * size ** 3))
        got["grad_" + name] = g
    return got


def _exact_attention(s, case):
    tokens, keys = _lengths(case)
    heads, kv, scale = case["heads"], case["kv_heads"], case["dim"] ** -0.5
    group = heads // kv
    grad = case["kind"] == "attention_grad"
    like = torch.zeros_like
    double = torch.float64
    got = {"grad_q": like(s["q"], dtype=double), "grad_k": like(s["k"], dtype=double),
           "grad_v": like(s["v"], dtype=double)} if grad else \
        {"out": like(s["q"], dtype=double), "lse": torch.full(s["q"].shape[:-1], -math.inf, dtype=double, device=DEVICE)}
    first = 0
    for b, (n, m) in enumerate(zip(tokens, keys)):
        if case["layout"] == "packed":
            at = key_at = slice(first, first + n)
            first += n
        else:
            at, key_at = (b, slice(0, n)), (b, slice(0, m))
        q, k, v = s["q"][at].double(), s["k"][key_at].double(), s["v"][key_at].double()
        last = torch.arange(n, device=DEVICE)[:, None] + (m - n)
        key = torch.arange(m, device=DEVICE)
        hidden = torch.zeros(n, m, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            hidden |= key > last
        if case["window"]:
            hidden |= key <= last - case["window"]
        g = s["grad_out"][at].double() if grad else None
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            scores = (q[:, h] * scale) @ kh.t()
            scores[hidden] = -math.inf
            lse = torch.logsumexp(scores, 1)
            p = scores.sub_(torch.where(lse.isinf(), 0.0, lse)[:, None]).exp_()
            if not grad:
                got["out"][at][:, h] = p @ vh
                got["lse"][at][:, h] = lse
                continue
            gh = g[:, h]
            got["grad_v"][key_at][:, h // group] += p.t() @ gh
            d = p * (gh @ vh.t() - (gh * (p @ vh)).sum(1, keepdim=True))
            got["grad_q"][at][:, h] = d @ kh * scale
            got["grad_k"][key_at][:, h // group] += d.t() @ q[:, h] * scale
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotary(s, case) if case["kind"] in ("rotary", "rotary_grad") else _exact_attention(s, case)
