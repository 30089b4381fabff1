"""Layer normalisation for training: the forward pass with kept statistics and the backward pass, against the formulas in fp64, and the
gradients against finite differences of the fp64 function.

Tolerances.  fp32: a row's sums of N terms are taken in fp32 by up to 16 terms a thread and a tree, so a statistic is off by at most
~(16 + 14) * 2^-24 < 2e-6 of the sum of magnitudes; y and dx are a handful of such factors, and values here are O(1): 1e-5 of the largest
value.  fp16: the same, then one rounding of at most half a step, 2^-11 relative to each value.  Column sums of R rows: at most R additions in
a chain, R * 2^-24 of the sum of magnitudes, written out in the test."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1.0e-6


def reference(x, ext, w, b, dy):
    x, dy = x.double(), dy.double()
    s = x if ext is None else x + ext.double()
    n = s.shape[-1]
    m = s.mean(-1, keepdim=True)
    r = 1 / (EPS + ((s - m) ** 2).sum(-1, keepdim=True) / (n - 1)).sqrt()
    xh = (s - m) * r
    g = dy if w is None else dy * w.double()
    y = xh * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).sum(-1, keepdim=True) / (n - 1))
    return y, torch.cat([m, r], -1), dx, dy * xh, dy


def make(seed, rows, channels, dtype, scale=1.0, offset=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, channels), device="cuda", generator=gen) * scale + offset).to(dtype)


def run(ctx, x, ext, w, b, dy, grad_dtype, beta_dx=0.0, beta_dw=0.0, dx=None, dw=None, db=None, y=None):
    from minml_b200 import backend as B
    rows, channels = x.shape
    y = torch.full_like(x, float("nan")) if y is None else y
    stats = torch.full((rows, 2), float("nan"), device="cuda")
    dx = torch.full_like(x, float("nan")) if dx is None else dx
    dw = torch.full((channels,), float("nan"), device="cuda", dtype=grad_dtype) if dw is None else dw
    db = torch.full((channels,), float("nan"), device="cuda", dtype=grad_dtype) if db is None else db
    B.layernormForwardTraining(ctx, x, y, w, b, stats, ext)
    ws = torch.full((max(1, B.layernormBackwardGetWorkspaceSize(ctx, x.shape)),), 255, device="cuda", dtype=torch.uint8)
    B.layernormBackward(ctx, x, dy, dx, w, stats, dw, db, ext=ext, beta_dx=beta_dx, beta_dw=beta_dw, workspace=ws)
    ctx.synchronize()
    return y, stats, dx, dw, db


def near(got, want, dtype, magnitude=None):
    magnitude = want.abs().max().clamp(min=1e-30) if magnitude is None else magnitude
    allowed = 1e-5 * magnitude + (2.0 ** -11 * want.abs() + 2.0 ** -25 if dtype == torch.float16 else 0.0)
    off = (got.double() - want).abs()
    assert bool((off <= allowed).all()), float((off - allowed).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("with_ext", [False, True])
@pytest.mark.parametrize("rows,channels", [
    (1, 2), (3, 7), (225, 256), (1000, 255), (17, 512), (5, 513), (64, 1000), (40, 1024), (9, 1025), (33, 2048), (7, 2052), (12, 4096), (5, 4097),
    (6, 8192), (3, 8193), (4, 20001), (20000, 40)])
def test_against_fp64(ctx, dtype, with_ext, rows, channels):
    x = make(1, rows, channels, dtype, 1.5, 0.25)
    ext = make(2, rows, channels, dtype) if with_ext else None
    w, b, dy = make(3, 1, channels, dtype, 0.3, 1.0)[0], make(4, 1, channels, dtype, 0.2)[0], make(5, rows, channels, dtype)
    y, stats, dx, dw, db = run(ctx, x, ext, w, b, dy, torch.float32)
    wy, ws, wdx, dw_terms, db_terms = reference(x, ext, w, b, dy)
    near(y, wy, dtype)
    near(stats, ws, torch.float32)
    near(dx, wdx, dtype, magnitude=(ws[:, 1:] * dy.double().abs().amax(1, keepdim=True) * 4).clamp(min=1e-30))
    for got, terms in ((dw, dw_terms), (db, db_terms)):
        assert bool(((got.double() - terms.sum(0)).abs() <= (rows + 32) * 2.0 ** -24 * terms.abs().sum(0) + 1e-5 * terms.abs().amax(0) + 1e-30).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("channels", [256, 1000, 4096])
def test_accumulation_in_place_and_gradient_types(ctx, dtype, channels):
    rows = 50
    x, dy, old = make(1, rows, channels, dtype), make(2, rows, channels, dtype), make(3, rows, channels, dtype)
    dw0, db0 = make(4, 1, channels, dtype)[0], make(5, 1, channels, dtype)[0]
    _, ws, wdx, tw, tb = reference(x, None, None, None, dy)
    y, _, dx, dw, db = run(ctx, x, None, None, None, dy, dtype, 0.5, 2.0, old.clone(), dw0.clone(), db0.clone())
    near(y, reference(x, None, None, None, dy)[0], dtype)
    near(dx, wdx + 0.5 * old.double(), dtype, magnitude=torch.tensor(20.0, device="cuda"))
    near(dw, tw.sum(0) + 2.0 * dw0.double(), dtype, magnitude=tw.abs().sum(0).max())
    near(db, tb.sum(0) + 2.0 * db0.double(), dtype, magnitude=tb.abs().sum(0).max())
    # y over x, dx over dy: the same bits as out of place
    from minml_b200 import backend as B
    x2, dy2, stats = x.clone(), dy.clone(), torch.empty((rows, 2), device="cuda")
    B.layernormForwardTraining(ctx, x2, x2, None, None, stats)
    ws = torch.empty(B.layernormBackwardGetWorkspaceSize(ctx, x.shape), device="cuda", dtype=torch.uint8)
    B.layernormBackward(ctx, x, dy2, dy2, None, stats, workspace=ws)
    ctx.synchronize()
    assert torch.equal(x2, y)
    want = torch.empty_like(dy)
    B.layernormBackward(ctx, x, dy, want, None, stats, workspace=ws)
    ctx.synchronize()
    assert torch.equal(dy2, want)


def test_offset_rows_and_unaligned_storage(ctx):
    """A large common offset must not cost the variance its digits, and rows that start on 2-byte boundaries take the narrow accesses."""
    for dtype, offset, scale in ((torch.float32, 1000.0, 1.0), (torch.float16, 100.0, 4.0)):
        storage = make(1, 1, 64 * 256 + 1, dtype, scale, offset)[0]
        x = storage[1:].view(64, 256)
        dy = make(2, 64, 256, dtype)
        y, stats, dx, dw, db = run(ctx, x, None, None, None, dy, torch.float32)
        wy, ws, wdx, tw, tb = reference(x, None, None, None, dy)
        # x - mean loses the offset's digits: (offset + |mean error|) * 2^-23 over the standard deviation
        slack = offset * 2.0 ** -22 / scale
        assert float((y.double() - wy).abs().max()) <= slack * 4 + 1e-5 * 4 + (2.0 ** -11 * 5 if dtype == torch.float16 else 0)
        assert float((dx.double() - wdx).abs().max()) <= (slack * 8 + 4e-5 + (2.0 ** -11 * 5 if dtype == torch.float16 else 0)) / scale


def test_constant_row_infinities_and_nan_stay_in_their_row(ctx):
    x, dy = make(1, 8, 512, torch.float32), make(2, 8, 512, torch.float32)
    x[1] = 3.0  # variance zero: r = 1 / sqrt(eps), everything finite
    x[3, 5] = float("inf")
    x[5, 7] = float("nan")
    y, stats, dx, dw, db = run(ctx, x, None, None, None, dy, torch.float32)
    wy, ws, wdx, _, _ = reference(x, None, None, None, dy)
    for r in (0, 2, 4, 6, 7):
        near(y[r], wy[r], torch.float32)
        near(dx[r], wdx[r], torch.float32, magnitude=torch.tensor(20.0, device="cuda"))
    assert float(y[1].abs().max()) == 0.0 and abs(float(stats[1, 1]) - 1000.0) <= 0.01
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[5]).all()) and bool(torch.isnan(dw).all())


def test_no_rows(ctx):
    from minml_b200 import backend as B
    x = torch.empty((0, 64), device="cuda", dtype=torch.float16)
    stats, dw, db = torch.empty((0, 2), device="cuda"), torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    B.layernormForwardTraining(ctx, x, x.clone(), None, None, stats)
    B.layernormBackward(ctx, x, x.clone(), x.clone(), None, stats, dw, db, beta_dw=0.5)
    ctx.synchronize()
    assert torch.equal(dw, torch.full_like(dw, 0.5)) and torch.equal(db, torch.full_like(db, 0.5))


def test_gradients_against_differences():
    """The formulas the kernels are tested against, in fp64, against central differences (no GPU result is involved)."""
    torch.manual_seed(0)
    x, w, b, dy = (torch.randn(s, dtype=torch.float64) for s in ((3, 9), (9,), (9,), (3, 9)))
    y, _, dx, tw, tb = reference(x, None, w, b, dy)
    h = 1e-5

    def f(x, w, b):
        return float((reference(x, None, w, b, dy)[0] * dy).sum())
    for t, grad, place in ((x, dx, 0), (w, tw.sum(0), 1), (b, tb.sum(0), 2)):
        for i in range(t.numel()):
            args = [x.clone(), w.clone(), b.clone()]
            args[place].view(-1)[i] += h
            up = f(*args)
            args[place].view(-1)[i] -= 2 * h
            assert abs((up - f(*args)) / (2 * h) - float(grad.reshape(-1)[i])) <= 1e-7


@pytest.mark.parametrize("rows,channels", [(225, 256), (300, 4096)])
def test_same_bits_every_time_and_in_a_graph(ctx, rows, channels):
    from minml_b200 import backend as B
    x, dy = make(1, rows, channels, torch.float16), make(2, rows, channels, torch.float16)
    first = run(ctx, x, None, None, None, dy, torch.float32)
    second = run(ctx, x, None, None, None, dy, torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    y, stats, dx, dw, db = (torch.empty_like(t) for t in first)
    ws = torch.empty(B.layernormBackwardGetWorkspaceSize(ctx, x.shape), device="cuda", dtype=torch.uint8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        B.layernormForwardTraining(ctx, x, y, None, None, stats)
        B.layernormBackward(ctx, x, dy, dx, None, stats, dw, db, workspace=ws)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, (y, stats, dx, dw, db)))


def test_refusals(ctx):
    from minml_b200 import backend as B
    x, stats = make(1, 8, 64, torch.float16), torch.empty((8, 2), device="cuda")
    y, ws = torch.empty_like(x), torch.empty(1 << 20, device="cuda", dtype=torch.uint8)
    dw = torch.empty(64, device="cuda")

    def forward(**k):
        a = dict(x=x, y=y, weights=None, bias=None, stats=stats)
        a.update(k)
        B.layernormForwardTraining(ctx, a["x"], a["y"], a["weights"], a["bias"], a["stats"], a.get("ext"))

    def backward(**k):
        a = dict(x=x, dy=y, dx=torch.empty_like(x), weights=None, stats=stats, dw=dw, db=dw.clone(), workspace=ws)
        a.update(k)
        B.layernormBackward(ctx, **a)
    cases = [
        (forward, dict(x=x.double(), y=y.double()), "fp16 or fp32"), (forward, dict(y=y.float()), "y is fp32"), (forward, dict(y=y[:7]), "y has"),
        (forward, dict(x=x[:, :1].contiguous(), y=y[:, :1].contiguous()), "at least 2 channels"), (forward, dict(weights=dw), "weights is fp32"),
        (forward, dict(bias=y[0, :32].contiguous()), "bias has"), (forward, dict(stats=stats[:4]), "stats has"), (forward, dict(ext=y[:4]), "ext has"),
        (forward, dict(y=x.view(-1)[64:].view(7, 64)), "y has"), (forward, dict(y=None), "y has rank 0"),
        (backward, dict(workspace=None), "needs a workspace"), (backward, dict(workspace=ws[:8]), "are needed"), (backward, dict(workspace=ws[8:]), "aligned"),
        (backward, dict(dw=dw.half()), "db is fp32"), (backward, dict(dw=dw.int()), "weight gradients"), (backward, dict(dy=y[:4]), "dy has"),
        (backward, dict(dw=dw, db=dw), "db overlaps dw"), (backward, dict(stats=None), "stats has rank 0")]
    for call, change, text in cases:
        with pytest.raises(B.BackendError, match=text):
            call(**change)
    wide = make(1, 2, 9000, torch.float16)
    with pytest.raises(B.BackendError, match="in place"):
        B.layernormForwardTraining(ctx, wide, wide, None, None, torch.empty((2, 2), device="cuda"))
    buf = torch.empty(9 * 64, device="cuda", dtype=torch.float16)
    with pytest.raises(B.BackendError, match="y overlaps x"):
        B.layernormForwardTraining(ctx, buf[:512].view(8, 64), buf[64:].view(8, 64), None, None, stats)
    forward()  # the context is usable after refusals
    backward()
    ctx.synchronize()
