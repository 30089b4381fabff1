"""Softmax cross entropy over a large vocabulary, forward and backward, against the formulas in fp64 with a forward error analysis
(error_bounds.py): logits and the running sums are fp32; fp16 rounds 2^15 P, the weighted rows of x and the results."""
import pytest
import torch

from tests.error_bounds import Bounded, product

pytestmark = pytest.mark.gpu


def make(seed, tokens, embed, vocab, dtype, ignored=0.2, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((tokens, embed), device="cuda", generator=gen).to(dtype)
    w = (torch.randn((vocab, embed), device="cuda", generator=gen) * spread * embed ** -0.5).to(dtype)
    targets = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
    skip = torch.rand(tokens, device="cuda", generator=gen) < ignored
    return x, w, torch.where(skip, torch.full_like(targets, -1), targets), torch.rand(tokens, device="cuda", generator=gen) * 2 - 0.5


def forward(x, w, targets):
    """loss and lse (Bounded) and the logits"""
    z = product(Bounded(x), Bounded(w).T, x.dtype)
    lse = torch.logsumexp(z.value, 1)
    # the sum of exponentials: each good to a few units and |z - max| 2^-23, hundreds of additions; lse itself rounded to fp32
    dlse = z.error.amax(1) + ((z.value.amax(1, keepdim=True) - z.value).amax(1) + 600) * 2.0 ** -23 + (lse.abs() + 20) * 2.0 ** -22
    valid = (targets >= 0) & (targets < w.shape[0])
    at = targets.long().clamp(0, w.shape[0] - 1)[:, None]
    loss = torch.where(valid, lse - z.value.gather(1, at)[:, 0], torch.zeros_like(lse))
    dloss = torch.where(valid, dlse + z.error.gather(1, at)[:, 0] + loss.abs() * 2.0 ** -23, torch.zeros_like(lse))
    return Bounded(loss, dloss), Bounded(lse, dlse), z, valid, at


def backward(x, w, targets, alpha, weights=None):
    dtype = x.dtype
    loss, lse, z, valid, at = forward(x, w, targets)
    c = valid.double() if weights is None else valid.double() * weights.double()
    p = torch.exp(z.value - lse.value[:, None])
    dp = p * (z.error + lse.error[:, None] + (z.value.abs() + lse.value.abs()[:, None] + 8) * 2.0 ** -22)
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    p = Bounded(p - hot, dp + hot * 2.0 ** -23)
    if dtype == torch.float16:
        p = Bounded(p.value, p.error + p.value.abs() * 2.0 ** -11 + 2.0 ** -40)
    p = Bounded(p.value * (c != 0).double()[:, None], p.error * (c != 0).double()[:, None])
    dx = product(p, Bounded(w), dtype).scaled(alpha * c[:, None])
    xw = Bounded(torch.where(c[:, None] != 0, x.double(), torch.zeros_like(x.double())) * c[:, None])
    if weights is not None and dtype == torch.float16:  # rounded as c / max |c| times x
        xw = Bounded(xw.value, xw.value.abs() * 2.0 ** -10 + 2.0 ** -25 * c.abs().max())
    return dx, product(p.T, xw.slack(2.0 ** -22), dtype).scaled(alpha)


def run(ctx, x, w, targets, alpha=1.0, weights=None, bytes_of_workspace=None, beta_dx=0.0, beta_dw=0.0, dx=None, dw=None):
    from minml_b200 import backend as B
    tokens = x.shape[0]
    loss, lse = (torch.full((tokens,), float("nan"), device="cuda") for _ in range(2))
    dx = torch.full_like(x, float("nan")) if dx is None else dx
    dw = torch.full_like(w, float("nan")) if dw is None else dw
    sizes = [B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, x.dtype, t) for t in (False, True)]
    if bytes_of_workspace is not None:
        sizes = bytes_of_workspace
    B.softmaxCrossEntropyForward(ctx, x, w, targets, loss, lse, torch.full((sizes[0],), 255, device="cuda", dtype=torch.uint8))
    B.softmaxCrossEntropyBackward(ctx, x, w, targets, lse, dx, dw, alpha, row_weights=weights, beta_dx=beta_dx, beta_dw=beta_dw,
                                  workspace=torch.full((sizes[1],), 255, device="cuda", dtype=torch.uint8))
    ctx.synchronize()
    return loss, lse, dx, dw


SIZES = [(1, 64, 1), (1, 256, 1000), (2, 128, 257), (7, 64, 5000), (16, 264, 700), (33, 128, 513), (64, 256, 4096), (65, 72, 999), (129, 256, 2000), (300, 512, 1025), (513, 128, 777),
         (1, 67, 301), (5, 33, 64), (70, 65, 1001)]


@pytest.mark.parametrize("tokens,embed,vocab", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("weighted", [False, True])
def test_against_fp64(ctx, dtype, weighted, tokens, embed, vocab):
    x, w, targets, weights = make(tokens + vocab, tokens, embed, vocab, dtype, 0.0 if tokens == 1 else 0.2)
    weights = weights if weighted else None
    if weighted and tokens > 3:
        weights[2] = 0.0
    alpha = 64.0
    want_loss, want_lse, *_ = forward(x, w, targets)
    want_dx, want_dw = backward(x, w, targets, alpha, weights)
    loss, lse, dx, dw = run(ctx, x, w, targets, alpha, weights)
    want_loss.holds(loss)
    want_lse.holds(lse)
    want_dx.holds(dx, dtype)
    want_dw.holds(dw, dtype)
    # accumulation
    old_x, old_w = torch.full_like(x, 0.5), torch.full_like(w, -0.5)
    _, _, dx, dw = run(ctx, x, w, targets, alpha, weights, beta_dx=2.0, beta_dw=0.5, dx=old_x.clone(), dw=old_w.clone())
    (want_dx + Bounded(old_x).scaled(2.0)).holds(dx, dtype)
    (want_dw + Bounded(old_w).scaled(0.5)).holds(dw, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_narrow_pieces(ctx, dtype):
    """The least workspace: pieces of 256 columns, the last one narrower."""
    from minml_b200 import backend as B
    x, w, targets, weights = make(3, 100, 128, 1100, dtype)
    least = []
    for training in (False, True):
        low, high = 0, B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, dtype, training)

        def fits(n):
            lse, loss = torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")
            ws = torch.empty(n, device="cuda", dtype=torch.uint8)
            try:
                if training:
                    B.softmaxCrossEntropyBackward(ctx, x, w, targets, lse, torch.empty_like(x), torch.empty_like(w), workspace=ws)
                else:
                    B.softmaxCrossEntropyForward(ctx, x, w, targets, loss, lse, ws)
            except B.BackendError:
                return False
            return True
        while high - low > 256:
            middle = (low + high) // 2
            low, high = (low, middle) if fits(middle) else (middle, high)
        least.append(high)
    want_loss, want_lse, *_ = forward(x, w, targets)
    want_dx, want_dw = backward(x, w, targets, 32.0, weights)
    loss, lse, dx, dw = run(ctx, x, w, targets, 32.0, weights, least)
    want_loss.holds(loss)
    want_lse.holds(lse)
    want_dx.holds(dx, dtype)
    want_dw.holds(dw, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens", [3, 140])
def test_rows_left_out_may_hold_anything(ctx, dtype, tokens):
    """Targets outside the vocabulary on both sides, and rows of weight 0: NaN and infinities there reach nothing else."""
    x, w, targets, weights = make(9, tokens, 128, 600, dtype, 0.0)
    clean = x.clone()
    targets[0], targets[1] = -7, 600
    weights[2] = 0.0
    clean[:3] = 1.0
    want_dx, want_dw = backward(clean, w, targets, 16.0, weights)
    x[0], x[1], x[2] = float("nan"), float("inf"), float("nan")
    loss, lse, dx, dw = run(ctx, x, w, targets, 16.0, weights)
    assert float(loss[0]) == 0.0 and float(loss[1]) == 0.0 and bool(torch.isnan(loss[2]))
    assert float(dx[:3].abs().max()) == 0.0
    if tokens > 3:
        Bounded(want_dx.value[3:], want_dx.error[3:]).holds(dx[3:], dtype)
    want_dw.holds(dw, dtype)


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("embed,vocab", [(516, 3001), (1030, 77), (2049, 5), (33, 9000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_few_tokens_of_any_row_length(ctx, dtype, embed, vocab, tokens):
    from minml_b200 import backend as B
    x, w, targets, _ = make(tokens + vocab, tokens, embed, vocab, dtype)
    targets[-1] = vocab - 1
    want_loss, want_lse, *_ = forward(x, w, targets)
    around = torch.full((2, tokens + 2), 7.0, device="cuda")
    loss, lse = around[0, 1:-1], around[1, 1:-1]
    size = B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, dtype, False)
    B.softmaxCrossEntropyForward(ctx, x, w, targets, loss, lse, torch.full((size,), 255, device="cuda", dtype=torch.uint8))
    ctx.synchronize()
    want_loss.holds(loss)
    want_lse.holds(lse)
    assert bool((around[:, 0] == 7.0).all()) and bool((around[:, -1] == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,embed,vocab", [(3, 64, 700), (3, 66, 700), (40, 64, 700), (140, 64, 700)])
def test_targets_at_the_ends_of_their_type(ctx, dtype, tokens, embed, vocab):
    """The least and the largest int32 are outside the vocabulary like any other such value: no arithmetic on them may come round to a column."""
    x, w, targets, _ = make(5, tokens, embed, vocab, dtype, 0.0)
    targets[0], targets[-1] = -2 ** 31, 2 ** 31 - 1
    want_loss, want_lse, *_ = forward(x, w, targets)
    want_dx, want_dw = backward(x, w, targets, 16.0)
    loss, lse, dx, dw = run(ctx, x, w, targets, 16.0)
    want_loss.holds(loss)
    want_lse.holds(lse)
    want_dx.holds(dx, dtype)
    want_dw.holds(dw, dtype)
    assert float(loss[0]) == 0.0 and float(loss[-1]) == 0.0 and not bool(dx[0].any()) and not bool(dx[-1].any())


def test_no_row_takes_part(ctx):
    x, w, targets, _ = make(9, 130, 64, 300, torch.float16, 2.0)
    assert int(targets.max()) == -1
    loss, lse, dx, dw = run(ctx, x, w, targets)
    assert float(loss.abs().max()) == 0.0 and float(dx.abs().max()) == 0.0 and float(dw.abs().max()) == 0.0


@pytest.mark.parametrize("tokens", [2, 200])
def test_large_logits(ctx, tokens):
    """Logits of hundreds: the maximum is taken out before the exponential, a certain row has loss 0 and a small gradient."""
    x, w, targets, _ = make(5, tokens, 64, 800, torch.float16, 0.0, spread=100.0)
    targets[0] = int((x[0].double() @ w.double().T).argmax())
    want_loss, want_lse, *_ = forward(x, w, targets)
    loss, lse, dx, dw = run(ctx, x, w, targets)
    want_loss.holds(loss)
    want_lse.holds(lse)
    want_dx, want_dw = backward(x, w, targets, 1.0)
    want_dx.holds(dx, torch.float16)
    want_dw.holds(dw, torch.float16)


def test_small_probabilities_keep_their_digits(ctx):
    """A probability far below fp16's normal range still gives its row of dW to fp16 precision."""
    tokens, embed, vocab = 130, 64, 4096
    x, w, targets, _ = make(6, tokens, embed, vocab, torch.float16, 0.0, spread=0.5)
    targets[:] = 0
    alpha = 4096.0
    _, want_dw = backward(x, w, targets, alpha)
    _, _, _, dw = run(ctx, x, w, targets, alpha)
    off = (dw[1:].double() - want_dw.value[1:]).norm() / want_dw.value[1:].norm()
    assert float(off) <= 2.0 ** -11 * 1.5  # two roundings of at most half a step each, in quadrature over many values


def test_no_tokens(ctx):
    from minml_b200 import backend as B
    x, w, targets, _ = make(1, 0, 64, 100, torch.float16)
    empty, dw = torch.empty(0, device="cuda"), torch.full_like(w, 2.0)
    B.softmaxCrossEntropyForward(ctx, x, w, targets, empty, empty.clone())
    B.softmaxCrossEntropyBackward(ctx, x, w, targets, empty, x.clone(), dw, beta_dw=0.5)
    ctx.synchronize()
    assert torch.equal(dw, torch.ones_like(w))


def test_the_formulas_against_differences():
    torch.manual_seed(2)
    x, w = torch.randn((4, 3), dtype=torch.float64), torch.randn((6, 3), dtype=torch.float64)
    targets, c = torch.tensor([1, -1, 5, 0], dtype=torch.int32), torch.tensor([0.5, 1.0, -2.0, 1.0], dtype=torch.float32)

    def f(x, w):
        z = x @ w.T
        keep = targets >= 0
        return float((c.double() * (torch.logsumexp(z, 1) - z.gather(1, targets.long().clamp(min=0)[:, None])[:, 0]))[keep].sum())
    dx, dw = backward(x, w, targets, 1.0, c)
    for t, grad, place in ((x, dx.value, 0), (w, dw.value, 1)):
        for i in range(t.numel()):
            args = [x.clone(), w.clone()]
            args[place].view(-1)[i] += 1e-5
            up = f(*args)
            args[place].view(-1)[i] -= 2e-5
            assert abs((up - f(*args)) / 2e-5 - float(grad.reshape(-1)[i])) <= 1e-7


@pytest.mark.parametrize("tokens,embed,vocab", [(1, 256, 3000), (200, 256, 3000)])
def test_same_bits_and_captured(ctx, tokens, embed, vocab):
    from minml_b200 import backend as B
    x, w, targets, weights = make(4, tokens, embed, vocab, torch.float16, 0.0)
    first = run(ctx, x, w, targets, 8.0, weights)
    assert all(torch.equal(a, b) for a, b in zip(first, run(ctx, x, w, targets, 8.0, weights)))
    out = [torch.full_like(t, float("nan")) for t in first]
    ws = torch.empty(B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, x.dtype, True), device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        B.softmaxCrossEntropyForward(ctx, x, w, targets, out[0], out[1], ws)
        B.softmaxCrossEntropyBackward(ctx, x, w, targets, out[1], out[2], out[3], 8.0, row_weights=weights, workspace=ws)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(out, first):
        assert torch.equal(got, want)


def test_refusals(ctx):
    from minml_b200 import backend as B
    x, w, targets, weights = make(1, 40, 64, 300, torch.float16)
    loss, lse = torch.zeros(40, device="cuda"), torch.zeros(40, device="cuda")
    ws = torch.empty(B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, x.dtype, True), device="cuda", dtype=torch.uint8)

    def fwd(**k):
        a = dict(x=x, weights=w, targets=targets, loss=loss, lse=lse, workspace=ws)
        a.update(k)
        B.softmaxCrossEntropyForward(ctx, **a)

    def bwd(**k):
        a = dict(x=x, weights=w, targets=targets, lse=lse, dx=torch.empty_like(x), dw=torch.empty_like(w), workspace=ws)
        a.update(k)
        B.softmaxCrossEntropyBackward(ctx, **a)
    for call, change, text in [
            (fwd, dict(x=x.double()), "fp16 or fp32"), (fwd, dict(weights=w.float()), "weights is fp32"), (fwd, dict(weights=w[:, :32].contiguous()), "x has|weights"),
            (fwd, dict(targets=targets[:39]), "targets has"), (fwd, dict(targets=targets.float()), "targets is fp32"), (fwd, dict(loss=loss.half()), "loss is fp16"),
            (fwd, dict(lse=loss), "lse overlaps loss"), (fwd, dict(workspace=None), "needs a workspace"), (fwd, dict(workspace=ws[:1024]), "are needed"),
            (bwd, dict(lse=None), "lse has rank 0"), (bwd, dict(dx=x), "dx overlaps x"), (bwd, dict(dw=w), "dw overlaps weights"), (bwd, dict(dw=torch.empty_like(x)), "dw has"),
            (bwd, dict(row_weights=weights[:4]), "row_weights has"), (bwd, dict(workspace=ws[:1024]), "are needed"), (bwd, dict(workspace=ws[2:]), "aligned")]:
        with pytest.raises(B.BackendError, match=text):
            call(**change)
    fwd()
    bwd()
    ctx.synchronize()
