"""Branches of the training operators that ordinary sizes take and the other tests' smaller ones do not: clusters of eight, a second accumulator in the
paired statistics kernel, sums of K ranges that several pieces of the vocabulary add to, and matrices of more than 2^31 elements."""
import pytest
import torch

from tests import test_gpu_cross_entropy as loss_tests
from tests import test_gpu_feed_forward as block_tests
from tests import test_gpu_layernorm_training as norm_tests

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 17, 48, 64])
@pytest.mark.parametrize("embed,hidden", [(512, 4096), (1000, 8200), (4104, 72)])
def test_clusters_of_eight(ctx, embed, hidden, tokens):
    """K from 4096 on with few weight rows: eight CTAs share them, each a range of K."""
    from minml_b200 import backend as B
    x, w1, w2, old = block_tests.make(tokens + hidden, tokens, embed, hidden, torch.float16)
    _, want, *_ = block_tests.forward(x, w1, w2, "silu")
    y = old.clone()
    B.gatedFeedForwardForward(ctx, x, w1, w2, y, "silu", beta=0.5, workspace=block_tests.workspace(ctx, x, w1, False))
    ctx.synchronize()
    (want + block_tests.Bounded(old).scaled(0.5)).holds(y, torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,embed,vocab", [(130, 2100, 3000), (65, 4096, 300)])
def test_loss_over_a_long_embed(ctx, dtype, tokens, embed, vocab):
    x, w, targets, weights = loss_tests.make(7, tokens, embed, vocab, dtype)
    loss, lse, dx, dw = loss_tests.run(ctx, x, w, targets, 64.0, weights)
    want_loss, want_lse, *_ = loss_tests.forward(x, w, targets)
    want_dx, want_dw = loss_tests.backward(x, w, targets, 64.0, weights)
    want_loss.holds(loss)
    want_lse.holds(lse)
    want_dx.holds(dx, dtype)
    want_dw.holds(dw, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens", [3, 70])
@pytest.mark.parametrize("share", [0.95, 0.75, 0.6, 0.45, 0.35])
def test_pieces_that_are_cut_along_k(ctx, dtype, tokens, share):
    """Few tokens, and a workspace for pieces of 500 to 1500 of 3000 columns: each piece's share of dx is cut into ranges of K, whose sums the next pieces add
    to, the last of them narrower and in fewer ranges."""
    from minml_b200 import backend as B
    x, w, targets, weights = loss_tests.make(11, tokens, 128, 3000, dtype)
    full = [B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, dtype, t) for t in (False, True)]
    sizes = [full[0] if dtype == torch.float16 or tokens < 17 else int(full[0] * share), int(full[1] * share)]
    old_x = torch.full_like(x, 0.25)
    try:
        _, _, dx, dw = loss_tests.run(ctx, x, w, targets, 32.0, weights, sizes, beta_dx=2.0, dx=old_x.clone())
    except B.BackendError as e:  # parts of the workspace that do not depend on the pieces
        assert "are needed" in str(e) and share < 0.7
        return
    want_dx, want_dw = loss_tests.backward(x, w, targets, 32.0, weights)
    (want_dx + loss_tests.Bounded(old_x).scaled(2.0)).holds(dx, dtype)
    want_dw.holds(dw, dtype)


# ------------------------------------------------------------------------------------------------ more than 2^31 elements
def ends(n, count=40):
    """the first, some middle and the last rows"""
    at = torch.cat([torch.arange(count), torch.linspace(0, n - 1, count).long(), torch.arange(n - count, n)])
    return at.unique().cuda()


def test_layer_norm_of_many_elements(ctx):
    from minml_b200 import backend as B
    rows, channels = (1 << 21) + 5, 1032
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((rows, channels), device="cuda", dtype=torch.float16).normal_(generator=gen)
    dy = torch.empty_like(x).normal_(generator=gen)
    y, dx, stats, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty((rows, 2), device="cuda"), torch.empty(channels, device="cuda"), torch.empty(channels, device="cuda")
    ws = torch.empty(B.layernormBackwardGetWorkspaceSize(ctx, x.shape), device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    B.layernormForwardTraining(ctx, x, y, None, None, stats)
    B.layernormBackward(ctx, x, dy, dx, None, stats, dw, db, workspace=ws)
    ctx.synchronize()
    at = ends(rows)
    wy, wstats, wdx, _, _ = norm_tests.reference(x[at], None, None, None, dy[at])
    norm_tests.near(y[at], wy, torch.float16)
    norm_tests.near(stats[at], wstats, torch.float32)
    norm_tests.near(dx[at], wdx, torch.float16, magnitude=(wstats[:, 1:] * dy[at].double().abs().amax(1, keepdim=True) * 4))
    sums, sizes = [torch.zeros(channels, device="cuda", dtype=torch.float64) for _ in range(2)], [torch.zeros(channels, device="cuda", dtype=torch.float64) for _ in range(2)]
    for first in range(0, rows, 1 << 18):
        part = slice(first, first + (1 << 18))
        _, _, _, tw, tb = norm_tests.reference(x[part], None, None, None, dy[part])
        for s, a, t in zip(sums, sizes, (tw, tb)):
            s += t.sum(0)
            a += t.abs().sum(0)
    # a thread's chain is rows / (blocks * teams), a few thousand rows at most, then the joining of blocks
    for got, s, a in zip((dw, db), sums, sizes):
        assert bool(((got.double() - s).abs() <= 2.0 ** 13 * 2.0 ** -24 * a).all())
    del x, y, dx, dy
    torch.cuda.empty_cache()


def test_gated_block_of_many_elements(ctx):
    from minml_b200 import backend as B
    tokens, embed, hidden = 2200000, 64, 1000  # h has 2.2e9 elements, [da du] 4.4e9
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((tokens, embed), device="cuda", dtype=torch.float16).normal_(generator=gen)
    dy = torch.empty_like(x).normal_(generator=gen)
    _, w1, w2, _ = block_tests.make(1, 1, embed, hidden, torch.float16)
    y, dx, dw1, dw2 = (torch.full_like(t, float("nan")) for t in (x, x, w1, w2))
    ws = torch.empty(B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, x.dtype, True, False), device="cuda", dtype=torch.uint8)
    assert ws.numel() > 3 * 2 ** 32
    torch.cuda.synchronize()
    B.gatedFeedForwardForward(ctx, x, w1, w2, y, "silu", workspace=ws)
    B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, dx, dw1, dw2, "silu", beta_dw=0.0, workspace=ws)
    ctx.synchronize()
    del ws
    at = ends(tokens)
    want_y, want_dx, _, _ = block_tests.backward(x[at], w1, w2, dy[at], "silu")
    want_y.holds(y[at], torch.float16)
    want_dx.holds(dx[at], torch.float16)
    sums = [torch.zeros_like(t, dtype=torch.float64) for t in (w1, w2)]
    for first in range(0, tokens, 100000):
        part = slice(first, first + 100000)
        xd, d = x[part].double(), dy[part].double()
        a, u = (xd @ w1.double().T).chunk(2, 1)
        v, slope = block_tests.act("silu", a)
        dh = d @ w2.double()
        sums[0] += torch.cat([dh * u * slope, dh * v], 1).T @ xd
        sums[1] += d.T @ (v * u)
    # every term's factor is rounded to fp16 once, 2^-11 at most, independently: in the sum's 2-norm 2^-11 of the terms' 2-norm; the result once more
    for got, want in zip((dw1, dw2), sums):
        assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -10
    torch.cuda.empty_cache()


def test_loss_of_many_elements(ctx):
    """dx has more than 2^31 elements in rows of odd length, so its sums are walked one element at a time with 64-bit places."""
    from minml_b200 import backend as B
    tokens, embed, vocab = 4200000, 513, 12
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((tokens, embed), device="cuda", dtype=torch.float16).normal_(generator=gen)
    w = (torch.randn((vocab, embed), device="cuda", generator=gen) * 2 * embed ** -0.5).half()
    targets = torch.randint(-1, vocab, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
    loss, lse, dx, dw = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    ws = torch.empty(B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, x.dtype, True), device="cuda", dtype=torch.uint8)
    alpha = 0.25
    torch.cuda.synchronize()
    B.softmaxCrossEntropyForward(ctx, x, w, targets, loss, lse, ws)
    B.softmaxCrossEntropyBackward(ctx, x, w, targets, lse, dx, dw, alpha, workspace=ws)
    ctx.synchronize()
    del ws
    at = ends(tokens)
    want_loss, want_lse, *_ = loss_tests.forward(x[at], w, targets[at])
    want_dx, _ = loss_tests.backward(x[at], w, targets[at], alpha)
    want_loss.holds(loss[at])
    want_lse.holds(lse[at])
    want_dx.holds(dx[at], torch.float16)
    total = torch.zeros_like(w, dtype=torch.float64)
    for first in range(0, tokens, 100000):
        part = slice(first, first + 100000)
        xd, t = x[part].double(), targets[part].long()
        p = torch.softmax(xd @ w.double().T, 1)
        p[torch.arange(t.numel(), device="cuda"), t.clamp(min=0)] -= 1
        total += alpha * (p * (t >= 0).double()[:, None]).T @ xd
    assert float((dw.double() - total).norm() / total.norm()) <= 2.0 ** -10
    torch.cuda.empty_cache()
