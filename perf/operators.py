"""What is measured of the operators for training and serving transformer blocks: layer normalisation with its backward pass, the
gated feed-forward block, and softmax cross entropy over a large vocabulary.

Where `own` is false, `run` computes plain forms from elementary torch operations in fp32; where it is true it makes the calls a
user makes of minml_b200.backend.  `exact` computes the same results in fp64 from the definitions, gradients by automatic
differentiation.
"""
import math

import torch

own = False

EPS = 1.0e-6  # inside the square root of the layer norm
TYPES = {"fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------------ cases
def _norm(name, rows, channels, dtype, ext):
    return {"name": name, "op": "norm", "rows": rows, "channels": channels, "dtype": dtype, "ext": ext}


def _ffn(name, tokens, embed, hidden, gate, dtype, train):
    return {"name": name, "op": "ffn", "tokens": tokens, "embed": embed, "hidden": hidden, "gate": gate, "dtype": dtype, "train": train}


def _loss(name, tokens, embed, vocab, dtype, train, ignored, weighted):
    return {"name": name, "op": "loss", "tokens": tokens, "embed": embed, "vocab": vocab, "dtype": dtype, "train": train, "ignored": ignored,
            "weighted": weighted}


def listed():
    return [
        # one board of 225 tokens with embed 256: the smallest training call, where the launches are what is paid for
        _norm("norm 225x256 fp16", 225, 256, "fp16", False),
        # the tokens of a language-model training batch, the residual sum fused into the norm
        _norm("norm 8192x4096 fp16 ext", 8192, 4096, "fp16", True),
        # fp32 training, odd sizes: rows that start on 4-byte boundaries only
        _norm("norm 4099x1001 fp32", 4099, 1001, "fp32", False),
        # decoding: one token, the weights are what is read
        _ffn("ffn 1 token fp16", 1, 4096, 11008, "silu", "fp16", False),
        # decoding a batch of sequences
        _ffn("ffn 48 tokens fp16", 48, 2048, 8192, "gelu", "fp16", False),
        # the benchmark's attention block (256 boards of 225 tokens, embed 256, hidden 1024) trained with a gated block
        _ffn("ffn 57600x256 fp16 train", 57600, 256, 1024, "silu", "fp16", True),
        # a language-model training batch
        _ffn("ffn 8192x4096 fp16 train", 8192, 4096, 11008, "silu", "fp16", True),
        # fp32 training, sizes that are multiples of nothing
        _ffn("ffn 777x517 fp32 train", 777, 517, 1363, "gelu", "fp32", True),
        # scoring one token against the whole vocabulary
        _loss("loss 1 token fp16", 1, 2048, 50021, "fp16", False, 0.0, False),
        # evaluation: a prompt's tokens scored, some of them padding
        _loss("loss 500x2048 fp16", 500, 2048, 50021, "fp16", False, 0.1, False),
        # a language-model training batch, a quarter of the rows masked out (a prompt, padding)
        _loss("loss 4096x4096 fp16 train", 4096, 4096, 100003, "fp16", True, 0.25, False),
        # fp32 training with a weight for every row
        _loss("loss 301x387 fp32 train", 301, 387, 8191, "fp32", True, 0.1, True),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], uniform in its logarithm; half of them rounded to a multiple of 64 where that leaves room."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n >= 128 and rng.random() < 0.5:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["norm", "ffn", "loss"])
    dtype = rng.choice(["fp16", "fp16", "fp32"])
    if op == "norm":
        channels = _spread(rng, 64, 8192)
        rows = _spread(rng, 1, min(60000, (1 << 25) // channels))
        c = _norm("", rows, channels, dtype, rng.random() < 0.5)
    elif op == "ffn":
        train = rng.random() < 0.5
        embed = _spread(rng, 128, 4096)
        hidden = _spread(rng, 128, 11008)
        most = int(min(60000, 3e11 / (embed * hidden))) // (1 if dtype == "fp16" else 8)
        tokens = _spread(rng, 1, max(1, most) if train else min(max(1, most), 4096))
        # relu in fp16 only: its derivative jumps at zero, and which side a pre-activation of 1e-7 falls on is rounding, not the operator
        c = _ffn("", tokens, embed, hidden, rng.choice(["sigmoid", "silu", "gelu"] + (["relu"] if dtype == "fp16" else [])), dtype, train)
    else:
        embed = _spread(rng, 64, 4096)
        vocab = _spread(rng, 500, 100000)
        most = int(min(8192, 1.2e12 / (embed * vocab))) // (1 if dtype == "fp16" else 8)
        c = _loss("", _spread(rng, 1, max(1, most)), embed, vocab, dtype, rng.random() < 0.5, rng.choice([0.0, 0.1, 0.5]), rng.random() < 0.3)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------------------ inputs
def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "norm":
        rows, channels = case["rows"], case["channels"]
        s["x"] = _normal(gen, (rows, channels), dtype, 1.5)
        s["ext"] = _normal(gen, (rows, channels), dtype) if case["ext"] else None
        s["w"] = (1 + 0.2 * torch.randn(channels, device="cuda", generator=gen)).to(dtype)
        s["b"] = _normal(gen, (channels,), dtype, 0.2)
        s["dy"] = _normal(gen, (rows, channels), dtype)
        s["y"], s["dx"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        s["stats"] = torch.empty((rows, 2), device="cuda")
        s["dw"], s["db"] = torch.empty(channels, device="cuda"), torch.empty(channels, device="cuda")
    elif case["op"] == "ffn":
        tokens, embed, hidden = case["tokens"], case["embed"], case["hidden"]
        s["x"] = _normal(gen, (tokens, embed), dtype)  # the output of a norm
        s["w1"] = _normal(gen, (2 * hidden, embed), dtype, embed ** -0.5)
        s["w2"] = _normal(gen, (embed, hidden), dtype, hidden ** -0.5)
        s["y"] = torch.empty((tokens, embed), device="cuda", dtype=dtype)
        if case["train"]:
            s["dy"] = _normal(gen, (tokens, embed), dtype)
            s["saved"] = torch.empty((tokens, 2 * hidden), device="cuda")
            s["dx"], s["dw1"], s["dw2"] = torch.empty_like(s["x"]), torch.empty_like(s["w1"]), torch.empty_like(s["w2"])
    else:
        tokens, embed, vocab = case["tokens"], case["embed"], case["vocab"]
        s["x"] = _normal(gen, (tokens, embed), dtype)
        s["w"] = _normal(gen, (vocab, embed), dtype, 2.0 * embed ** -0.5)  # logits of standard deviation 2
        targets = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
        skip = torch.rand(tokens, device="cuda", generator=gen) < case["ignored"]
        s["targets"] = torch.where(skip, torch.full_like(targets, -1), targets)
        s["weights"] = torch.rand(tokens, device="cuda", generator=gen) + 0.5 if case["weighted"] else None
        s["alpha"] = 65536.0 / tokens  # the mean over the tokens times the loss scale that keeps fp16 gradients in range
        s["loss"], s["lse"] = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda")
        if case["train"]:
            s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["w"])
    s["workspace"] = {}
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(s):
    x = s["x"].float()
    if s["ext"] is not None:
        x = x + s["ext"].float()
    n = x.shape[1]
    centred = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt(EPS + (centred * centred).sum(1, keepdim=True) / (n - 1))
    xh = centred * r
    w, dy = s["w"].float(), s["dy"].float()
    y = xh * w + s["b"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - xh * ((g * xh).sum(1, keepdim=True) / (n - 1)))
    return {"y": y.to(s["x"].dtype), "dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0)}


def _gate(kind, g):
    """act(g) and act'(g)"""
    if kind == "relu":
        return torch.clamp(g, min=0.0), (g > 0).to(g.dtype)
    if kind == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    sig = 1.0 / (1.0 + torch.exp(-g))
    if kind == "sigmoid":
        return sig, sig * (1.0 - sig)
    return g * sig, sig * (1.0 + g * (1.0 - sig))


def _plain_ffn(s):
    dtype, hidden = s["x"].dtype, s["hidden"]
    x, w1, w2 = s["x"].float(), s["w1"].float(), s["w2"].float()
    gu = x @ w1.T
    u = gu[:, hidden:]
    a, da = _gate(s["gate"], gu[:, :hidden])
    h = a * u
    out = {"y": (h @ w2.T).to(dtype)}
    if s["train"]:
        dy = s["dy"].float()
        dh = dy @ w2
        dgu = torch.cat([dh * u * da, dh * a], 1)
        out.update(dx=(dgu @ w1).to(dtype), dw1=(dgu.T @ x).to(dtype), dw2=(dy.T @ h).to(dtype))
    return out


def _plain_loss(s):
    dtype, targets = s["x"].dtype, s["targets"].long()
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.T
    top = z.max(1, keepdim=True).values
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    valid = targets >= 0
    at = targets.clamp(min=0)[:, None]
    out = {"loss": torch.where(valid, (lse - z.gather(1, at))[:, 0], torch.zeros_like(lse[:, 0]))}
    if s["train"]:
        scale = valid.float() * s["alpha"]
        if s["weights"] is not None:
            scale = scale * s["weights"]
        p = torch.exp(z - lse)
        p.scatter_add_(1, at, -torch.ones_like(lse))
        p = p * scale[:, None]
        out.update(dx=(p @ w).to(dtype), dw=(p.T @ x).to(dtype))
    return out


# ------------------------------------------------------------------------------------------------------------------ the framework's calls
_user = {}


def _framework():
    """The backend module and one context, as a user's program holds them."""
    if not _user:
        from minml_b200 import backend
        _user["backend"], _user["ctx"] = backend, backend.Context(torch.cuda.current_device())
    return _user["backend"], _user["ctx"]


def _workspace(s, nbytes):
    """The state's scratch tensor, made on its first pass."""
    if "buffer" not in s["workspace"]:
        s["workspace"]["buffer"] = torch.empty(max(1, nbytes), device="cuda", dtype=torch.uint8)
    return s["workspace"]["buffer"]


def _own_norm(s):
    B, ctx = _framework()
    B.layernormForwardTraining(ctx, s["x"], s["y"], s["w"], s["b"], s["stats"], s["ext"])
    ws = _workspace(s, B.layernormBackwardGetWorkspaceSize(ctx, s["x"].shape))
    B.layernormBackward(ctx, s["x"], s["dy"], s["dx"], s["w"], s["stats"], s["dw"], s["db"], ext=s["ext"], workspace=ws)
    return {"y": s["y"], "dx": s["dx"], "dw": s["dw"], "db": s["db"]}


def _own_ffn(s):
    B, ctx = _framework()
    if "buffer" not in s["workspace"]:
        _workspace(s, B.gatedFeedForwardGetWorkspaceSize(ctx, s["x"].shape, s["w1"].shape, s["x"].dtype, s["train"]))
    ws = s["workspace"]["buffer"]
    B.gatedFeedForwardForward(ctx, s["x"], s["w1"], s["w2"], s["y"], s["gate"], saved=s["saved"] if s["train"] else None, workspace=ws)
    out = {"y": s["y"]}
    if s["train"]:
        B.gatedFeedForwardBackward(ctx, s["x"], s["w1"], s["w2"], s["dy"], s["dx"], s["dw1"], s["dw2"], s["gate"], saved=s["saved"], workspace=ws)
        out.update(dx=s["dx"], dw1=s["dw1"], dw2=s["dw2"])
    return out


def _own_loss(s):
    B, ctx = _framework()
    if "buffer" not in s["workspace"]:
        _workspace(s, B.softmaxCrossEntropyGetWorkspaceSize(ctx, s["x"].shape, s["w"].shape, s["x"].dtype, s["train"]))
    ws = s["workspace"]["buffer"]
    B.softmaxCrossEntropyForward(ctx, s["x"], s["w"], s["targets"], s["loss"], s["lse"], workspace=ws)
    out = {"loss": s["loss"]}
    if s["train"]:
        B.softmaxCrossEntropyBackward(ctx, s["x"], s["w"], s["targets"], s["lse"], s["dx"], s["dw"], s["alpha"], row_weights=s["weights"], workspace=ws)
        out.update(dx=s["dx"], dw=s["dw"])
    return out


def run(state):
    op = state["op"]
    if own:
        return _own_norm(state) if op == "norm" else _own_ffn(state) if op == "ffn" else _own_loss(state)
    return _plain_norm(state) if op == "norm" else _plain_ffn(state) if op == "ffn" else _plain_loss(state)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    es = 2 if case["dtype"] == "fp16" else 4
    if case["op"] == "norm":
        # x (and the summand) and dy read, y and dx written; weights, bias and their gradients
        n = case["rows"] * case["channels"]
        return {"bytes": n * es * (5 if case["ext"] else 4) + case["channels"] * (2 * es + 8), "flops": 20 * n}
    if case["op"] == "ffn":
        t, d, f = case["tokens"], case["embed"], case["hidden"]
        weights, rows = 3 * d * f, t * d
        if case["train"]:  # x, dy, weights in; y, dx, weight gradients out
            return {"bytes": es * (4 * rows + 2 * weights), "flops": 18 * t * d * f}
        return {"bytes": es * (2 * rows + weights), "flops": 6 * t * d * f}
    t, d, v = case["tokens"], case["embed"], case["vocab"]
    if case["train"]:  # logits, then dx and dw from them
        return {"bytes": es * (2 * t * d + 2 * v * d) + 8 * t, "flops": 6 * t * d * v}
    return {"bytes": es * (t * d + v * d) + 8 * t, "flops": 2 * t * d * v}


# ------------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    leaf = lambda t: t.double().requires_grad_(case.get("train", True))  # noqa: E731
    x = leaf(s["x"])
    if case["op"] == "norm":
        w, b = leaf(s["w"]), leaf(s["b"])
        full = x if s["ext"] is None else x + s["ext"].double()
        y = (full - full.mean(1, keepdim=True)) / (full.var(1, unbiased=True, keepdim=True) + EPS).sqrt() * w + b
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if case["op"] == "ffn":
        w1, w2 = leaf(s["w1"]), leaf(s["w2"])
        g, u = torch.nn.functional.linear(x, w1).chunk(2, 1)
        act = {"relu": torch.relu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}[case["gate"]]
        y = torch.nn.functional.linear(act(g) * u, w2)
        out = {"y": y.detach()}
        if case["train"]:
            out.update(zip(("dx", "dw1", "dw2"), torch.autograd.grad(y, (x, w1, w2), s["dy"].double())))
        return out
    w = leaf(s["w"])
    loss = torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w), s["targets"].long(), ignore_index=-1, reduction="none")
    out = {"loss": loss.detach()}
    if case["train"]:
        scale = torch.full_like(loss, s["alpha"]) if s["weights"] is None else s["alpha"] * s["weights"].double()
        out.update(zip(("dx", "dw"), torch.autograd.grad(loss, (x, w), scale)))
    return out
