"""The training operators together, as a step of a pre-norm block with a loss uses them:
   n1 = LN1(a);  b = a + FFN(n1);  n2 = LN2(b);  loss = mean CE(n2 W^T),
forward and backward through the layer classes, against automatic differentiation in fp64 of the same network.

Tolerances, relative in the 2-norm.  fp16: every activation and every gradient that is handed on is rounded once, by at most 2^-11 relative
to each value; a result has at most seven such roundings behind it (n1, h, b, n2, 2^15 P, the rounded gradients on the way back, itself), and no
step here amplifies a relative error by more than two: 7 * 2 * 2^-11 < 7e-3.  fp32: sums of at most a few thousand terms, a few 1e-6."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def build(ctx, dtype, embed, hidden, vocab, gate="silu"):
    from minml_b200 import layers as L
    r = np.random.default_rng(embed + vocab)

    def n(*shape, scale=1.0, offset=0.0):
        return (r.standard_normal(shape) * scale + offset).astype(np.float32)
    net = {
        "ln1": L.LayerNormalization(ctx, n(embed, scale=0.1, offset=1.0), n(embed, scale=0.1), dtype),
        "ffn": L.GatedFeedForward(ctx, n(2 * hidden, embed, scale=embed ** -0.5), n(embed, hidden, scale=hidden ** -0.5), gate, dtype),
        "ln2": L.LayerNormalization(ctx, n(embed, scale=0.1, offset=1.0), n(embed, scale=0.1), dtype),
        "head": L.SoftmaxCrossEntropy(ctx, n(vocab, embed, scale=2 * embed ** -0.5), dtype)}
    return net


def step(ctx, net, a, targets, alpha, saved):
    """One forward and backward pass; every buffer is made here, as a program makes them once at its start."""
    from minml_b200 import layers as L
    tokens, embed = a.shape
    ffn, head = net["ffn"], net["head"]
    ws = L.Workspace(ctx)
    ws.reserve(max(net["ln1"].backward_workspace_bytes(a.shape), ffn.workspace_bytes(a.shape, True, saved is not None), head.workspace_bytes(a.shape, True)))
    f32 = dict(device="cuda", dtype=torch.float32)
    n1, n2, b = (torch.empty_like(a) for _ in range(3))
    s1, s2 = torch.empty((tokens, 2), **f32), torch.empty((tokens, 2), **f32)
    loss, lse = torch.empty(tokens, **f32), torch.empty(tokens, **f32)
    b.copy_(a)
    torch.cuda.synchronize()
    net["ln1"].forward_training([a], n1, s1)
    ffn.forward([n1], b, ws, saved=saved, beta=1.0)
    net["ln2"].forward_training([b], n2, s2)
    head.forward([n2], targets, loss, ws, lse)
    dn2, db, dn1 = (torch.empty_like(a) for _ in range(3))
    dw, dw1, dw2 = torch.empty_like(head.weights), torch.empty_like(ffn.w1), torch.empty_like(ffn.w2)
    g1, h1, g2, h2 = (torch.empty(embed, **f32) for _ in range(4))
    head.backward([n2], targets, lse, dn2, dw, ws, alpha)
    net["ln2"].backward([b], s2, dn2, db, g2, h2, ws)
    ffn.backward([n1], db, dn1, dw1, dw2, ws, saved=saved)
    net["ln1"].backward([a], s1, dn1, db, g1, h1, ws, beta_prev=1.0)  # into the residual path's gradient: db becomes da
    return {"loss": loss, "da": db, "dw": dw, "dw1": dw1, "dw2": dw2, "dg1": g1, "db1": h1, "dg2": g2, "db2": h2}


def reference(net, a, targets, alpha):
    def leaf(t):
        return t.double().requires_grad_()
    leaves = {"da": leaf(a), "dw": leaf(net["head"].weights), "dw1": leaf(net["ffn"].w1), "dw2": leaf(net["ffn"].w2), "dg1": leaf(net["ln1"].gamma),
              "db1": leaf(net["ln1"].beta), "dg2": leaf(net["ln2"].gamma), "db2": leaf(net["ln2"].beta)}

    def norm(x, g, b):
        return (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=True, keepdim=True) + 1e-6).sqrt() * g + b
    p = leaves
    n1 = norm(p["da"], p["dg1"], p["db1"])
    g, u = (n1 @ p["dw1"].T).chunk(2, 1)
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[net["ffn"].gate]
    b = p["da"] + (act(g) * u) @ p["dw2"].T
    loss = torch.nn.functional.cross_entropy(norm(b, p["dg2"], p["db2"]) @ p["dw"].T, targets.long(), ignore_index=-1, reduction="none")
    grads = torch.autograd.grad((loss * alpha).sum(), list(leaves.values()))
    return dict(zip(leaves, grads), loss=loss.detach())


@pytest.mark.parametrize("tokens,embed,hidden,vocab", [(1, 128, 256, 500), (40, 256, 512, 1000), (450, 256, 1024, 1500), (300, 1152, 520, 700), (33, 100, 90, 301)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("keep", [True, False])
def test_training_step(ctx, dtype, keep, tokens, embed, hidden, vocab):
    net = build(ctx, dtype, embed, hidden, vocab, "silu" if keep else "gelu")
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    a = torch.randn((tokens, embed), device="cuda", generator=gen).to(dtype)
    targets = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
    if tokens > 1:
        targets[::5] = -1
    alpha = 1024.0 / tokens
    saved = torch.empty((tokens, 2 * hidden), device="cuda") if keep else None
    got = step(ctx, net, a, targets, alpha, saved)
    ctx.synchronize()
    for name, want in reference(net, a, targets, alpha).items():
        # the loss itself is fp32, but of an n2 that is rounded like the rest
        off = float((got[name].double() - want).norm() / want.norm())
        assert off <= (7e-3 if dtype == torch.float16 else 1e-5), (name, off)


def test_training_step_captured_and_on_a_board_shaped_tensor(ctx):
    """The whole step in one CUDA graph, replayed on changing inputs; [boards, h, w, embed] tensors are matrices of boards * h * w rows."""
    from minml_b200 import layers as L
    tokens, embed, hidden, vocab = 2 * 225, 256, 512, 700
    net = build(ctx, torch.float16, embed, hidden, vocab)
    ffn = net["ffn"]
    ws = L.Workspace(ctx)
    boards = torch.randn((2, 15, 15, embed), device="cuda").half()
    ws.reserve(ffn.workspace_bytes(boards.shape, True, False))
    y, dx, dw1, dw2 = torch.empty_like(boards), torch.empty_like(boards), torch.empty_like(ffn.w1), torch.empty_like(ffn.w2)
    dy = torch.randn_like(boards)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        ffn.forward([boards], y, ws)
        ffn.backward([boards], dy, dx, dw1, dw2, ws)
    for seed in (1, 2):
        boards.copy_(torch.randn((2, 15, 15, embed), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).half())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        flat = boards.view(tokens, embed)
        want = [torch.empty_like(t) for t in (flat, flat, ffn.w1, ffn.w2)]
        ffn.forward([flat], want[0], ws)
        ffn.backward([flat], dy.view(tokens, embed), want[1], want[2], want[3], ws)
        ctx.synchronize()
        for got, w in zip((y, dx, dw1, dw2), want):
            assert torch.equal(got.view(w.shape), w)
    del graph


def test_another_stream_of_torch(ctx):
    """Inputs made on a torch stream of their own: the context's stream is ordered behind it by wait_for_torch, results are read after synchronize."""
    from minml_b200 import backend as B
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = torch.randn((5000, 256), device="cuda").half()
        for _ in range(20):
            x = (x * 1.0).contiguous()
        y, stats = torch.empty_like(x), torch.empty((5000, 2), device="cuda")
        ctx.wait_for_torch()
        B.layernormForwardTraining(ctx, x, y, None, None, stats)
        ctx.synchronize()
        want = (x.double() - x.double().mean(1, keepdim=True)) / (x.double().var(1, keepdim=True) + 1e-6).sqrt()
    torch.cuda.synchronize()
    assert float((y.double() - want).abs().max()) <= 2.0 ** -11 * 6


def test_operands_of_another_device_or_layout_are_refused(ctx):
    from minml_b200 import backend as B
    x, stats = torch.zeros((8, 64), device="cuda", dtype=torch.float16), torch.empty((8, 2), device="cuda")
    with pytest.raises(B.BackendError, match="passed to a context"):
        B.layernormForwardTraining(ctx, x.cpu(), x, None, None, stats)
    with pytest.raises(B.BackendError, match="dense row-major"):
        B.layernormForwardTraining(ctx, torch.zeros((64, 8), device="cuda", dtype=torch.float16).T, x, None, None, stats)
    with pytest.raises(B.BackendError, match="fp16 or fp32"):
        B.layernormForwardTraining(ctx, x.bfloat16(), x, None, None, stats)
    w1, w2 = torch.zeros((32, 64), device="cuda", dtype=torch.float16), torch.zeros((64, 16), device="cuda", dtype=torch.float16)
    ws = torch.empty(1 << 20, device="cuda", dtype=torch.uint8)
    shifted = torch.zeros(8 * 64 + 1, device="cuda", dtype=torch.float16)[1:].view(8, 64)
    with pytest.raises(B.BackendError, match="x must be 16-byte aligned"):
        B.gatedFeedForwardForward(ctx, shifted, w1, w2, x.clone(), workspace=ws)
    loss = torch.empty(8, device="cuda")
    with pytest.raises(B.BackendError, match="x must be 16-byte aligned"):
        B.softmaxCrossEntropyForward(ctx, shifted, w1, torch.zeros(8, device="cuda", dtype=torch.int32), loss, None, ws)


def test_two_contexts_at_once():
    """Two contexts on one device, each with its own workspace, with nothing ordering their streams."""
    from minml_b200 import backend as B
    contexts = [B.Context(0), B.Context(0)]
    jobs = []
    for i, c in enumerate(contexts):
        gen = torch.Generator(device="cuda").manual_seed(i)
        x = torch.randn((700, 512), device="cuda", generator=gen).half()
        w = torch.randn((4000, 512), device="cuda", generator=gen).half() * 0.05
        t = torch.randint(0, 4000, (700,), device="cuda", generator=gen, dtype=torch.int32)
        ws = torch.empty(B.softmaxCrossEntropyGetWorkspaceSize(c, x.shape, w.shape, x.dtype, True), device="cuda", dtype=torch.uint8)
        jobs.append((c, x, w, t, ws, [torch.empty(700, device="cuda"), torch.empty(700, device="cuda"), torch.empty_like(x), torch.empty_like(w)]))
    torch.cuda.synchronize()

    def run(job):
        c, x, w, t, ws, out = job
        B.softmaxCrossEntropyForward(c, x, w, t, out[0], out[1], ws)
        B.softmaxCrossEntropyBackward(c, x, w, t, out[1], out[2], out[3], 64.0, workspace=ws)
    alone = []
    for job in jobs:
        run(job)
        job[0].synchronize()
        alone.append([o.clone() for o in job[-1]])
    torch.cuda.synchronize()
    for _ in range(5):
        for job in jobs:
            run(job)
    for job, want in zip(jobs, alone):
        job[0].synchronize()
        assert all(torch.equal(a, b) for a, b in zip(job[-1], want))
    for c in contexts:
        c.close()
