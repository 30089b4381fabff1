"""The gated feed-forward block, forward and backward, against the formulas in fp64 with a forward error analysis (error_bounds.py): the
roundings of fp16 are those of h, da and du and of the results; pre-activations are kept in fp32."""
import math

import pytest
import torch

from tests.error_bounds import Bounded, product

pytestmark = pytest.mark.gpu

GATES = ["sigmoid", "relu", "silu", "gelu"]
CURVATURE = {"sigmoid": 0.1, "relu": 0.0, "silu": 0.5, "gelu": 1.2}  # bounds of |act''|
SLOPE = {"sigmoid": 0.25, "relu": 1.0, "silu": 1.1, "gelu": 1.13}  # and of |act'|


def act(kind, g):
    if kind == "relu":
        return g.clamp(min=0), (g > 0).double()
    if kind == "gelu":
        phi = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if kind == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def forward(x, w1, w2, kind):
    """Bounded h and y, and what the backward pass needs"""
    dtype = x.dtype
    hidden = w1.shape[0] // 2
    au = product(Bounded(x), Bounded(w1).T, dtype)
    a, u = Bounded(au.value[:, :hidden], au.error[:, :hidden]), Bounded(au.value[:, hidden:], au.error[:, hidden:])
    v, d = act(kind, a.value)
    # the value of the activation in fp32: its exponential is good to |a| 2^-23 and a few units
    dv = a.error * SLOPE[kind] + (v.abs() + 1) * (a.value.abs() + 8) * 2.0 ** -23
    h = Bounded(v * u.value, dv * (u.value.abs() + u.error) + v.abs() * u.error).rounded(dtype)
    return h, product(h, Bounded(w2).T, dtype), a, u, v, dv, d


def backward(x, w1, w2, dy, kind):
    dtype = x.dtype
    h, y, a, u, v, dv, d = forward(x, w1, w2, kind)
    dh = product(Bounded(dy), Bounded(w2), dtype)
    dd = a.error * CURVATURE[kind] + (d.abs() + 1) * (a.value.abs() + 8) * 2.0 ** -23
    if kind == "relu":
        dd = dd + (a.value.abs() <= a.error).double()  # the derivative jumps where the pre-activation's sign is not certain
    ud = Bounded(u.value * d, u.error * (d.abs() + dd) + u.value.abs() * dd).slack(2.0 ** -23)
    da = Bounded(dh.value * ud.value, dh.error * (ud.value.abs() + ud.error) + dh.value.abs() * ud.error).slack(2.0 ** -23).rounded(dtype)
    du = Bounded(dh.value * v, dh.error * (v.abs() + dv) + dh.value.abs() * dv).slack(2.0 ** -23).rounded(dtype)
    dau = Bounded(torch.cat([da.value, du.value], 1), torch.cat([da.error, du.error], 1))
    return y, product(dau, Bounded(w1), dtype), product(dau.T, Bounded(x), dtype), product(Bounded(dy).T, h, dtype)


def make(seed, tokens, embed, hidden, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def n(shape, scale):
        return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)
    return n((tokens, embed), 1.0), n((2 * hidden, embed), embed ** -0.5), n((embed, hidden), hidden ** -0.5), n((tokens, embed), 1.0)


def workspace(ctx, x, w1, training, saved=True, poison=True):
    from minml_b200 import backend as B
    size = B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, x.dtype, training, saved)
    return torch.full((max(1, size),), 255 if poison else 0, device="cuda", dtype=torch.uint8)


def nan_like(t):
    return torch.full_like(t, float("nan"))


SIZES = [(1, 64, 64), (2, 256, 40), (5, 128, 1024), (9, 264, 136), (16, 64, 520), (17, 512, 256), (31, 104, 72), (48, 256, 512), (64, 128, 256), (65, 136, 264), (128, 256, 256),
         (200, 96, 88), (257, 256, 384), (300, 1104, 264), (64, 1032, 512), (300, 512, 1000), (700, 64, 128), (1025, 320, 264),
         (1, 67, 33), (3, 33, 130), (40, 35, 71), (130, 65, 129)]


@pytest.mark.parametrize("tokens,embed,hidden", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_forward(ctx, dtype, tokens, embed, hidden):
    from minml_b200 import backend as B
    x, w1, w2, old = make(tokens + embed, tokens, embed, hidden, dtype)
    for i, kind in enumerate(GATES):
        h, want, *_ = forward(x, w1, w2, kind)
        y = nan_like(x)
        ws = workspace(ctx, x, w1, False)
        B.gatedFeedForwardForward(ctx, x, w1, w2, y, kind, workspace=ws)
        ctx.synchronize()
        want.holds(y, dtype)
        if i == 2:  # the residual sum, and the training form of the forward pass
            y2 = old.clone()
            saved = torch.full((tokens, 2 * hidden), float("nan"), device="cuda")
            B.gatedFeedForwardForward(ctx, x, w1, w2, y2, kind, beta=0.5, saved=saved, workspace=workspace(ctx, x, w1, True))
            ctx.synchronize()
            (want + Bounded(old).scaled(0.5)).holds(y2, dtype)


@pytest.mark.parametrize("tokens,embed,hidden", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_backward(ctx, dtype, tokens, embed, hidden):
    from minml_b200 import backend as B
    x, w1, w2, dy = make(tokens + hidden, tokens, embed, hidden, dtype)
    for i, kind in enumerate(GATES):
        want_y, want_dx, want_dw1, want_dw2 = backward(x, w1, w2, dy, kind)
        for keep in (True, False):
            saved = torch.full((tokens, 2 * hidden), float("nan"), device="cuda") if keep else None
            ws = workspace(ctx, x, w1, True, keep)
            y, dx, dw1, dw2 = nan_like(x), nan_like(x), nan_like(w1), nan_like(w2)
            B.gatedFeedForwardForward(ctx, x, w1, w2, y, kind, saved=saved, workspace=ws)
            ws.fill_(255)  # nothing may be carried from one call to the next in the scratch memory
            B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, dx, dw1, dw2, kind, saved=saved, workspace=ws)
            ctx.synchronize()
            want_y.holds(y, dtype)
            want_dx.holds(dx, dtype)
            want_dw1.holds(dw1, dtype)
            want_dw2.holds(dw2, dtype)
    # accumulation, and gradients asked for one at a time
    old_x, old_1, old_2 = (torch.ones_like(t) * 0.25 for t in (x, w1, w2))
    dx, dw1, dw2 = old_x.clone(), old_1.clone(), old_2.clone()
    ws = workspace(ctx, x, w1, True, False)
    B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, dx, None, None, kind, beta_dx=2.0, workspace=ws)
    B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, None, dw1, None, kind, beta_dw=-1.0, workspace=ws)
    B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, None, None, dw2, kind, beta_dw=0.5, workspace=ws)
    ctx.synchronize()
    (want_dx + Bounded(old_x).scaled(2.0)).holds(dx, dtype)
    (want_dw1 + Bounded(old_1).scaled(-1.0)).holds(dw1, dtype)
    (want_dw2 + Bounded(old_2).scaled(0.5)).holds(dw2, dtype)


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("embed,hidden", [(516, 1028), (1030, 514), (2049, 131), (33, 2051)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_few_tokens_of_any_row_length(ctx, dtype, embed, hidden, tokens):
    """Rows read by fours, by twos and singly, short and shared by several warps; the memory around y is left as it was."""
    from minml_b200 import backend as B
    x, w1, w2, old = make(tokens + embed, tokens, embed, hidden, dtype)
    around = torch.full((tokens + 2, embed), 7.0, device="cuda", dtype=dtype)
    y = around.view(-1)[embed:-embed].view(tokens, embed)
    if y.data_ptr() % 16:  # (results need their element's alignment only)
        assert embed % 8
    for kind, beta in (("silu", 0.0), ("gelu", -1.5)):
        _, want, *_ = forward(x, w1, w2, kind)
        y.copy_(old)
        B.gatedFeedForwardForward(ctx, x, w1, w2, y, kind, beta=beta, workspace=workspace(ctx, x, w1, False))
        ctx.synchronize()
        (want if beta == 0.0 else want + Bounded(old).scaled(beta)).holds(y, dtype)
        assert bool((around[0] == 7.0).all()) and bool((around[-1] == 7.0).all())


@pytest.mark.parametrize("tokens,embed,hidden,dtype", [(1, 512, 1024, torch.float32), (5, 514, 1031, torch.float32), (16, 256, 512, torch.float32), (40, 256, 1000, torch.float32),
                                                       (3, 1001, 2000, torch.float16), (2, 512, 1024, torch.float16), (300, 264, 512, torch.float32)])
def test_calls_in_a_row_see_new_values(ctx, dtype, tokens, embed, hidden):
    """The same buffers with other contents in every call, launched back to back: no kernel may read what an earlier call left in a cache."""
    from minml_b200 import backend as B
    x, w1, w2, _ = make(tokens + embed, tokens, embed, hidden, dtype)
    gen = torch.Generator(device="cuda").manual_seed(3)
    inputs = [torch.randn(x.shape, device="cuda", generator=gen).to(dtype) for _ in range(12)]
    results = [nan_like(x) for _ in inputs]
    ws = workspace(ctx, x, w1, False)
    torch.cuda.synchronize()
    with torch.cuda.stream(ctx.torch_stream()):
        for i in range(len(inputs)):
            x.copy_(inputs[i])
            B.gatedFeedForwardForward(ctx, x, w1, w2, results[i], "gelu", workspace=ws)
    ctx.synchronize()
    for i in range(len(inputs)):
        forward(inputs[i], w1, w2, "gelu")[1].holds(results[i], dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_few_tokens_off_their_alignment(ctx, dtype):
    """Padded operands may begin at any element, also where their row length alone would allow wider reads."""
    from minml_b200 import backend as B
    tokens, embed, hidden = 3, 52 if dtype == torch.float16 else 50, 66
    x, w1, w2, _ = make(11, tokens, embed, hidden, dtype)
    _, want, *_ = forward(x, w1, w2, "silu")
    shifted = []
    for t in (x, w1, w2):
        buffer = torch.zeros(t.numel() + 1, device="cuda", dtype=dtype)
        buffer[1:] = t.view(-1)
        shifted.append(buffer[1:].view(t.shape))
    y = nan_like(x)
    B.gatedFeedForwardForward(ctx, *shifted, y, "silu", workspace=workspace(ctx, x, w1, False))
    ctx.synchronize()
    want.holds(y, dtype)


def test_the_formulas_against_differences():
    """act' and the backward formulas in fp64, against central differences of the forward formula."""
    torch.manual_seed(1)
    for kind in GATES:
        x, w1, w2, dy = (torch.randn(s, dtype=torch.float64) for s in ((3, 5), (8, 5), (5, 4), (3, 5)))

        def f(x, w1, w2):
            a, u = (x @ w1.T).chunk(2, 1)
            return float(((act(kind, a)[0] * u) @ w2.T * dy).sum())
        a, u = (x @ w1.T).chunk(2, 1)
        v, d = act(kind, a)
        dh = dy @ w2
        dau = torch.cat([dh * u * d, dh * v], 1)
        for t, grad, place in ((x, dau @ w1, 0), (w1, dau.T @ x, 1), (w2, dy.T @ (v * u), 2)):
            for i in range(t.numel()):
                args = [x.clone(), w1.clone(), w2.clone()]
                args[place].view(-1)[i] += 1e-5
                up = f(*args)
                args[place].view(-1)[i] -= 2e-5
                assert abs((up - f(*args)) / 2e-5 - float(grad.reshape(-1)[i])) <= 1e-6


def test_extreme_pre_activations(ctx):
    """Gates far out on both sides: no NaN from exp's overflow, and the limits of the activations."""
    from minml_b200 import backend as B
    tokens, embed, hidden = 130, 64, 128
    x = torch.zeros((tokens, embed), device="cuda", dtype=torch.float16)
    x[:, 0], x[:, 1] = 1.0, 1.0
    w1 = torch.zeros((2 * hidden, embed), device="cuda", dtype=torch.float16)
    w1[:hidden, 0] = torch.tensor([-6.0e4, -500.0, -90.0, -20.0, 0.0, 20.0, 90.0, 500.0] * 16, device="cuda")
    w1[hidden:, 1] = 1.0
    w2 = torch.zeros((embed, hidden), device="cuda", dtype=torch.float16)
    w2[:8, :8] = torch.eye(8, device="cuda")
    for kind in GATES:
        for t in (1, tokens):
            y, dx, dw1, dw2 = nan_like(x[:t]), nan_like(x[:t]), nan_like(w1), nan_like(w2)
            ws = workspace(ctx, x, w1, True, False)
            B.gatedFeedForwardForward(ctx, x[:t], w1, w2, y, kind, workspace=ws)
            B.gatedFeedForwardBackward(ctx, x[:t], w1, w2, torch.ones_like(x[:t]), dx, dw1, dw2, kind, workspace=ws)
            ctx.synchronize()
            want = act(kind, w1[:8, 0].double())[0]
            assert bool(((y[0, :8].double() - want).abs() <= want.abs() * 2.0 ** -9 + 1e-6).all())
            assert all(bool(torch.isfinite(g).all()) for g in (dx, dw1, dw2))


def test_nan_stays_in_its_token(ctx):
    from minml_b200 import backend as B
    x, w1, w2, dy = make(3, 150, 128, 136, torch.float16)
    h, want, *_ = forward(x, w1, w2, "silu")
    x[70, 3], x[1, 0] = float("nan"), float("inf")
    y = nan_like(x)
    B.gatedFeedForwardForward(ctx, x, w1, w2, y, workspace=workspace(ctx, x, w1, False))
    ctx.synchronize()
    clean = torch.ones(150, dtype=torch.bool, device="cuda")
    clean[70] = clean[1] = False
    assert bool(torch.isnan(y[70]).all()) and not bool(torch.isfinite(y[1]).any())
    Bounded(want.value[clean], want.error[clean]).holds(y[clean], torch.float16)


def test_no_tokens(ctx):
    from minml_b200 import backend as B
    x, w1, w2, dy = make(1, 0, 64, 72, torch.float16)
    dw1, dw2 = nan_like(w1), torch.ones_like(w2)
    B.gatedFeedForwardForward(ctx, x, w1, w2, x.clone())
    B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, x.clone(), dw1, None)
    B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, None, None, dw2, beta_dw=0.5)
    ctx.synchronize()
    assert float(dw1.abs().max()) == 0.0 and torch.equal(dw2, torch.full_like(dw2, 0.5))


@pytest.mark.parametrize("tokens,embed,hidden", [(1, 512, 1032), (24, 256, 512), (512, 256, 512), (300, 1280, 520)])
def test_same_bits_and_graphs_with_their_own_workspaces(ctx, tokens, embed, hidden):
    """Two graphs captured on one context, each with a workspace of its own, replayed on two streams at the same time."""
    from minml_b200 import backend as B
    sets = []
    for seed in (1, 2):
        x, w1, w2, dy = make(seed, tokens, embed, hidden, torch.float16)
        saved = torch.empty((tokens, 2 * hidden), device="cuda")
        sets.append((x, w1, w2, dy, saved, workspace(ctx, x, w1, True), [nan_like(t) for t in (x, x, w1, w2)]))

    def both(x, w1, w2, dy, saved, ws, out):
        B.gatedFeedForwardForward(ctx, x, w1, w2, out[0], "gelu", saved=saved, workspace=ws)
        B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, out[1], out[2], out[3], "gelu", saved=saved, workspace=ws)
    eager = []
    for s in sets:
        both(*s)
        ctx.synchronize()
        eager.append([t.clone() for t in s[-1]])
        both(*s)
        ctx.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager[-1], s[-1]))
    graphs = []
    for s in sets:
        for t in s[-1]:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=ctx.torch_stream()):
            both(*s)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, want in zip(sets, eager):
        assert all(torch.equal(a, b) for a, b in zip(s[-1], want))


@pytest.mark.parametrize("tokens,embed,hidden", [(1, 512, 1032), (7, 515, 700), (300, 260, 521), (1500, 128, 640)])
def test_fp32_same_bits_and_graphs_at_the_same_time(ctx, tokens, embed, hidden):
    """As above for fp32: pairs of CTAs, few rows and joined K ranges of two graphs share the device."""
    from minml_b200 import backend as B
    sets, graphs, want = [], [], []
    for seed in (1, 2):
        x, w1, w2, dy = make(seed, tokens, embed, hidden, torch.float32)
        sets.append((x, w1, w2, dy, torch.empty((tokens, 2 * hidden), device="cuda"), workspace(ctx, x, w1, True), [nan_like(t) for t in (x, x, w1, w2)]))

    def both(x, w1, w2, dy, saved, ws, out):
        B.gatedFeedForwardForward(ctx, x, w1, w2, out[0], "silu", saved=saved, workspace=ws)
        B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, out[1], out[2], out[3], "silu", saved=saved, workspace=ws)
    for s in sets:
        both(*s)
        ctx.synchronize()
        want.append([t.clone() for t in s[-1]])
        for t in s[-1]:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=ctx.torch_stream()):
            both(*s)
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(s[-1], w))


def test_refusals(ctx):
    from minml_b200 import backend as B
    x, w1, w2, dy = make(1, 40, 64, 72, torch.float16)
    ws = workspace(ctx, x, w1, True, False)
    saved = torch.empty((40, 144), device="cuda")

    def fwd(**k):
        a = dict(x=x, w1=w1, w2=w2, y=torch.empty_like(x), gate="silu", workspace=ws)
        a.update(k)
        B.gatedFeedForwardForward(ctx, **a)

    def bwd(**k):
        a = dict(x=x, w1=w1, w2=w2, dy=dy, dx=torch.empty_like(x), dw1=torch.empty_like(w1), dw2=torch.empty_like(w2), workspace=ws)
        a.update(k)
        B.gatedFeedForwardBackward(ctx, **a)
    for call, change, text in [
            (fwd, dict(x=x.double()), "fp16 or fp32"), (fwd, dict(w1=w1.float()), "w1 is fp32"), (fwd, dict(w2=w2.T.contiguous()), "w1 must be"), (fwd, dict(w1=w1[:143]), "w1 must be"),
            (fwd, dict(x=x[:, :32].contiguous()), "x has"), (fwd, dict(y=x), "y overlaps x"), (fwd, dict(y=torch.empty_like(dy[:39])), "y has"), (fwd, dict(gate="tanh"), "unknown gate"),
            (fwd, dict(workspace=None), "needs a workspace"), (fwd, dict(workspace=ws[:64]), "are needed"), (fwd, dict(workspace=ws[1:]), "aligned"),
            (fwd, dict(saved=saved.half()), "saved is fp16"), (fwd, dict(saved=saved[:, :72].contiguous()), "saved has"),
            (bwd, dict(dx=dy), "dx overlaps dy"), (bwd, dict(dw1=w1), "dw1 overlaps w1"), (bwd, dict(dw2=torch.empty_like(w1)), "dw2 has"), (bwd, dict(dy=dy.float()), "dy is fp32"),
            (bwd, dict(workspace=ws[:64]), "are needed"), (bwd, dict(workspace=None), "needs a workspace"), (bwd, dict(saved=saved[:3]), "saved has")]:
        with pytest.raises(B.BackendError, match=text):
            call(**change)
    fwd()
    bwd()
    ctx.synchronize()
