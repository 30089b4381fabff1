"""Gates far below zero under a large factor: a sigmoid that is zero to any digit of the result leaves nothing of u, however large u is."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gate", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("tokens", [1, 70, 300])
@pytest.mark.parametrize("embed,keep", [(64, False), (64, True), (1032, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_closed_gates_let_nothing_through(ctx, dtype, embed, keep, tokens, gate):
    """a = -4e5 to -4e4 and u = 4e5 to 4e4: act(a) and act'(a) are below e^-39000, so h, y, da, du and every gradient but for zeros' signs are zero."""
    from minml_b200 import backend as B
    hidden = 96
    x = torch.full((tokens, embed), 100.0, device="cuda", dtype=dtype)
    w1 = torch.full((2 * hidden, embed), 6400.0 / 64 * 0.6 * 64 / embed, device="cuda", dtype=dtype)
    w1[:hidden] *= -1
    w1 *= torch.linspace(0.1, 1.0, hidden, device="cuda").repeat(2)[:, None].to(dtype)
    w2 = torch.ones((embed, hidden), device="cuda", dtype=dtype)
    dy = torch.full_like(x, 3.0)
    a = float((x[:1].double() @ w1[:hidden].double().T).max())
    assert a < -3.0e4
    y, dx, dw1, dw2 = (torch.full_like(t, float("nan")) for t in (x, x, w1, w2))
    saved = torch.empty((tokens, 2 * hidden), device="cuda") if keep else None
    ws = torch.empty(B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, dtype, True, keep), device="cuda", dtype=torch.uint8)
    B.gatedFeedForwardForward(ctx, x, w1, w2, y, gate, saved=saved, workspace=ws)
    B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, dx, dw1, dw2, gate, saved=saved, workspace=ws)
    ctx.synchronize()
    for result in (y, dx, dw1, dw2):
        assert not bool(result.any()), float(result.double().abs().max())  # (a NaN counts)
