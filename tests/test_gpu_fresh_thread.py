"""Calls from a thread that has not used CUDA before: every entry point makes its context's device current before the driver is asked for anything."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def in_a_fresh_thread(call):
    errors = []

    def body():
        try:
            call()
        except Exception as e:
            errors.append(e)
    thread = threading.Thread(target=body)
    thread.start()
    thread.join()
    if errors:
        raise errors[0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 40, 200])
@pytest.mark.parametrize("what", ["block forward", "block backward", "loss forward", "loss backward", "norm"])
def test_the_training_operators(ctx, what, tokens, dtype):
    from minml_b200 import backend as B
    gen = torch.Generator(device="cuda").manual_seed(tokens)

    def n(*shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)
    embed, hidden, vocab = 64, 128, 500
    x, dy, w1, w2, w = n(tokens, embed), n(tokens, embed), n(2 * hidden, embed, scale=0.1), n(embed, hidden, scale=0.1), n(vocab, embed, scale=0.1)
    targets = torch.randint(0, vocab, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
    loss, lse, stats = torch.empty(tokens, device="cuda"), torch.full((tokens,), 8.0, device="cuda"), torch.empty((tokens, 2), device="cuda")
    size = max(B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, dtype, True, False), B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, w.shape, dtype, True))
    ws = torch.empty(size, device="cuda", dtype=torch.uint8)
    outs = {"block forward": [x], "block backward": [x, w1, w2], "loss forward": [loss], "loss backward": [x, w], "norm": [x]}[what]
    fresh, here = ([torch.full_like(t, float("nan")) for t in outs] for _ in range(2))
    calls = {"block forward": lambda o: B.gatedFeedForwardForward(ctx, x, w1, w2, o[0], workspace=ws), "block backward": lambda o: B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, *o, workspace=ws),
             "loss forward": lambda o: B.softmaxCrossEntropyForward(ctx, x, w, targets, o[0], None, ws), "loss backward": lambda o: B.softmaxCrossEntropyBackward(ctx, x, w, targets, lse, *o, workspace=ws),
             "norm": lambda o: B.layernormForwardTraining(ctx, x, o[0], None, None, stats)}
    torch.cuda.synchronize()
    in_a_fresh_thread(lambda: calls[what](fresh))
    ctx.synchronize()
    calls[what](here)
    ctx.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(fresh, here))


@pytest.mark.parametrize("channels", [64, 128, 256])
def test_convolutions_and_products(ctx, channels):
    from minml_b200 import layers as L
    r = np.random.default_rng(1)
    weights = (r.standard_normal((channels, 3, 3, channels)) * 0.05).astype(np.float32)
    x = torch.randn((3, 15, 15, channels), device="cuda").half()
    y = [torch.empty_like(x) for _ in range(4)]
    conv, dense = L.Conv2D(ctx, weights, None, "relu"), L.Conv2D(ctx, weights[:, 1:2, 1:2], None, "relu")
    ws = L.Workspace(ctx)
    ws.reserve(conv.workspace_bytes(x.shape))
    torch.cuda.synchronize()
    in_a_fresh_thread(lambda: conv.forward([x], y[0], ws))
    in_a_fresh_thread(lambda: dense.forward([x], y[1], None))
    ctx.synchronize()
    conv.forward([x], y[2], ws)
    dense.forward([x], y[3], None)
    ctx.synchronize()
    assert torch.equal(y[0], y[2]) and torch.equal(y[1], y[3])
