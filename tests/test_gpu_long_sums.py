"""Sums over many indices.  The tensor core cuts its fp32 sums where an addition would round, always toward zero: each step of a sum over n steps
loses up to 2^-23 of the sum so far.  Operands of one sign make such losses add up, so these tests see how long the library lets one accumulator
grow, which the elementwise bounds of the other tests do not."""
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
