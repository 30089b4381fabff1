"""fp32 products on pairs of SMs: whole numbers whose products and partial sums all fit fp32's 24 bits, so a result is exact or wrong.  The
weights have 13 bits, of which an operand's upper term holds 11: a lower term that belongs to another stage, or is not there yet, shows as a
difference of at least 1 in a sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(seed, tokens, embed, hidden):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def whole(shape, low, high, share):
        v = torch.randint(low, high + 1, shape, device="cuda", generator=gen).float()
        sign = torch.randint(0, 2, shape, device="cuda", generator=gen).float() * 2 - 1
        return v * sign * (torch.rand(shape, device="cuda", generator=gen) < share)
    x = whole((tokens, embed), 1, 2, 0.25)
    x[:, 0] = 1.0
    w1 = whole((2 * hidden, embed), 2 ** 12, 2 ** 13 - 1, 1.0)
    w1[:hidden] = 0.0
    w1[:hidden, 0] = 1.0  # a = 1, and relu lets h = u pass
    taken = torch.randint(0, hidden, (embed,), device="cuda", generator=gen)
    w2 = torch.zeros((embed, hidden), device="cuda")
    w2[torch.arange(embed, device="cuda"), taken] = 1.0  # y[t, n] = u[t, taken[n]]
    return x, w1, w2, whole((tokens, embed), 1, 2, min(0.02, 6.0 / tokens))


@pytest.mark.parametrize("tokens,embed,hidden", [(130, 4096, 512), (300, 1030, 263), (3000, 512, 384)])
def test_whole_numbers_over_many_stages(ctx, tokens, embed, hidden):
    from minml_b200 import backend as B
    rounds = 12
    limit = float(2 ** 24)
    x, w1, w2, dy = make(0, tokens, embed, hidden)
    saved = torch.empty((tokens, 2 * hidden), device="cuda")
    ws = torch.empty(B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, x.dtype, True), device="cuda", dtype=torch.uint8)
    inputs = [make(seed + 1, tokens, embed, hidden) for seed in range(rounds)]
    results = [[torch.full_like(t, float("nan")) for t in (x, x, w1, w2)] for _ in range(rounds)]
    torch.cuda.synchronize()
    with torch.cuda.stream(ctx.torch_stream()):  # the same buffers with other values in every round, back to back
        for values, (y, dx, dw1, dw2) in zip(inputs, results):
            for t, v in zip((x, w1, w2, dy), values):
                t.copy_(v)
            B.gatedFeedForwardForward(ctx, x, w1, w2, y, "relu", saved=saved, workspace=ws)
            B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, dx, dw1, dw2, "relu", saved=saved, workspace=ws)
    ctx.synchronize()
    for values, (y, dx, dw1, dw2) in zip(inputs, results):
        vx, v1, v2, vdy = (t.double() for t in values)
        u = vx @ v1[hidden:].T
        dh = vdy @ v2
        assert float((vx.abs() @ v1[hidden:].abs().T).max()) < limit and float((vdy.abs().T @ u.abs()).max()) < limit and float((dh.abs() @ v1[hidden:].abs()).max()) < limit
        assert torch.equal(y.double(), u @ v2.T)
        assert torch.equal(dx[:, 1:].double(), (dh @ v1[hidden:])[:, 1:])  # (column 0 also takes da Wg, which need not fit)
        assert torch.equal(dw1[hidden:].double(), dh.T @ vx)
        assert torch.equal(dw2.double(), vdy.T @ u)
