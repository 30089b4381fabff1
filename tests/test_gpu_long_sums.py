"""Sums over many indices.  The tensor core cuts its fp32 sums where an addition would round, always toward zero: each of two
groups of 8 terms in a step of 16 loses up to 2^-23 of the sum so far.  Operands of one sign make such losses add up, so these tests see how
long the library lets one accumulator grow, which the elementwise bounds of the other tests do not."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,embed", [(130, 4096), (130, 8200), (300, 2056)])
def test_a_certain_row_has_no_gradient(ctx, tokens, embed):
    """Every row's target is column 0 with a logit of 35 to 65 made of terms of one sign; the other logits are below 8, so 1 - P is below 1e-8.
    What is left of P - 1 is the rounding of lse, maximum plus logarithm, by 2^-24 relative, its product with log2 e by another 2^-24, and the
    exponent's argument (up to 17, half a step 2^-20) and power by 2^-20: 65 * 2^-23 + 2^-19 < 1e-5.  The logits lose digits of their own, but the
    same ones in the forward and the backward pass, if both sum up in the same segments."""
    from minml_b200 import backend as B
    vocab, alpha = 640, 1024.0
    gen = torch.Generator(device="cuda").manual_seed(embed)
    x = (torch.rand((tokens, embed), device="cuda", generator=gen) + 0.5).half()
    w = (torch.randn((vocab, embed), device="cuda", generator=gen) * embed ** -0.5).half()
    w[0] = ((torch.rand(embed, device="cuda", generator=gen) + 0.5) * (60.0 / embed)).half()
    x *= torch.linspace(0.6, 1.05, tokens, device="cuda")[:, None].half()
    targets = torch.zeros(tokens, device="cuda", dtype=torch.int32)
    z = x.double() @ w.double().T
    assert float(z[:, 0].max()) < 65 and float(z[:, 0].min()) > 35 and float(z[:, 1:].max()) < 8
    loss, lse = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ws = torch.empty(B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, x.dtype, True), device="cuda", dtype=torch.uint8)
    B.softmaxCrossEntropyForward(ctx, x, w, targets, loss, lse, ws)
    B.softmaxCrossEntropyBackward(ctx, x, w, targets, lse, dx, dw, alpha, workspace=ws)
    ctx.synchronize()
    p = torch.softmax(z, 1)
    p[:, 0] = -p[:, 1:].sum(1)  # P - 1
    off = (dx.double() - alpha * p @ w.double()).abs()
    allowed = alpha * 1e-5 * w[0].double().abs() + 2.0 ** -25 + 1e-6
    assert bool((off <= allowed).all()), float((off / allowed).max())
    off = (dw[0].double() - alpha * p[:, 0] @ x.double()).abs()
    allowed = alpha * 1e-5 * x.double().sum(0) + 2.0 ** -25
    assert bool((off <= allowed).all()), float((off / allowed).max())


def test_weight_gradients_over_many_tokens(ctx):
    """262 144 tokens whose terms all have one sign: 16 384 steps of 16 tokens, two cuts a step, would come out 16 384 / 2 * 2^-22 = 2e-3 low at
    most, and came out 1.7e-3 low.  The library sums at most 8 192 tokens an accumulator: 512 / 2 * 2^-22 = 6.1e-5 at most.  h, da, du and the
    results are rounded, which the mean over 16 x 256 results of 262 144 terms each leaves 2^-11 / 64 of at most: 8e-6.  (dw1 has 74 tiles, one for
    each pair of SMs, and dw2 half as many, cut into two ranges of tokens.)"""
    from minml_b200 import backend as B
    tokens, embed, hidden, some = 262144, 256, 9472, 16
    gen = torch.Generator(device="cuda").manual_seed(1)

    def positive(shape, scale):
        return ((torch.rand(shape, device="cuda", generator=gen) + 0.5) * scale).half()
    x, dy = positive((tokens, embed), 1.0), positive((tokens, embed), 2.0 ** -10)
    w1, w2 = positive((2 * hidden, embed), 1.0 / embed), positive((embed, hidden), 1.0 / embed)
    dx, dw1, dw2 = torch.empty_like(x), torch.empty_like(w1), torch.empty_like(w2)
    ws = torch.empty(B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, x.dtype, True, False), device="cuda", dtype=torch.uint8)
    B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, dx, dw1, dw2, "sigmoid", workspace=ws)
    ctx.synchronize()
    at = torch.linspace(0, hidden - 1, some, device="cuda").long()
    xd, dyd = x.double(), dy.double()
    s = torch.sigmoid(xd @ w1[at].double().T)
    u, dh = xd @ w1[hidden + at].double().T, dyd @ w2[:, at].double()
    wanted = ((dh * u * s * (1 - s)).T @ xd, dw1[at]), ((dh * s).T @ xd, dw1[hidden + at]), (dyd.T @ (s * u), dw2[:, at])
    for want, got in wanted:
        low = float((got.double() / want - 1).mean())
        assert abs(low) <= 6.1e-5 + 8e-6, low


@pytest.mark.parametrize("tokens", [1, 16, 20, 33, 49, 64, 65])
@pytest.mark.parametrize("embed", [1024, 5000, 16384])
def test_log_sum_of_rows_over_a_long_embed(ctx, embed, tokens):
    """One column of a row has a logit of 35 to 65 made of terms of one sign, so lse is that logit.  Accumulators take 1024 indices: 64 / 2 * 2^-22 =
    7.7e-6 of the sum at most; adding up to 16 of them rounds by 16 * 2^-24, and lse by a few 2^-23."""
    from minml_b200 import backend as B
    vocab = 300
    gen = torch.Generator(device="cuda").manual_seed(embed)
    x = (torch.rand((tokens, embed), device="cuda", generator=gen) + 0.5).half()
    w = (torch.randn((vocab, embed), device="cuda", generator=gen) * embed ** -0.5).half()
    w[0] = ((torch.rand(embed, device="cuda", generator=gen) + 0.5) * (60.0 / embed)).half()
    x *= torch.linspace(0.6, 1.05, tokens, device="cuda")[:, None].half()
    targets = torch.ones(tokens, device="cuda", dtype=torch.int32)
    loss, lse = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda")
    ws = torch.empty(B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, x.dtype), device="cuda", dtype=torch.uint8)
    B.softmaxCrossEntropyForward(ctx, x, w, targets, loss, lse, ws)
    ctx.synchronize()
    z = x.double() @ w.double().T
    want = torch.logsumexp(z, 1)
    assert float(want.min()) > 30 and float(z[:, 1:].max()) < 8
    assert float(((lse.double() - want).abs() / want).max()) <= 7.7e-6 + 16 * 2.0 ** -24 + 4 * 2.0 ** -23


def test_fp32_products_over_a_long_sum(ctx):
    """y = h W2^T with K = 8192 terms of one sign and h exact (the gate is 1, u picks elements of x, of 20 bits).  An accumulator takes 32 indices, 12
    instructions with two cuts of 2^-23 each at most: 12 * 2^-22; the dropped product of the lower terms is at most 2^-20 and their rounding 2^-21:
    4.4e-6 in all.  The 256 additions of fp32 round by half a step either way: in the mean over 2.4 million results nothing.  (74 tiles: one range of
    K.)  One accumulator for all of K would come out 1 024 * 3 / 2 * 2^-22 = 3.7e-4 low at most; 5.7e-5 was measured."""
    from minml_b200 import backend as B
    tokens, embed, hidden = 512, 4736, 8192
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(2 ** 18, 3 * 2 ** 18, (tokens, embed), device="cuda", generator=gen).float() * 2.0 ** -19
    x[:, 0] = 1.0
    taken = torch.randint(0, embed, (hidden,), device="cuda", generator=gen)
    w1 = torch.zeros((2 * hidden, embed), device="cuda")
    w1[:hidden, 0] = 1.0
    w1[hidden + torch.arange(hidden, device="cuda"), taken] = 1.0
    w2 = torch.rand((embed, hidden), device="cuda", generator=gen) + 0.5
    y = torch.empty_like(x)
    ws = torch.empty(B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, x.dtype), device="cuda", dtype=torch.uint8)
    B.gatedFeedForwardForward(ctx, x, w1, w2, y, "relu", workspace=ws)
    ctx.synchronize()
    off = y.double() / (x[:, taken].double() @ w2.double().T) - 1
    assert abs(float(off.mean())) <= 4.4e-6, float(off.mean())
    assert float(off.abs().max()) <= 4.4e-6 + 128 * 2.0 ** -24
