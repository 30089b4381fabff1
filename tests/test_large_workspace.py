"""Scratch memory beyond the 2^31 - 1 elements of a descriptor's extent: a flat tensor of bytes is what the size functions and Workspace lead to."""
import pytest
import torch


class Nowhere:
    """Stands for a context whose device is where CPU tensors say they are."""
    handle = None
    device_index = -1


def test_a_workspace_above_two_gigabytes_is_described():
    from minml_b200 import backend as B
    x, stats = torch.zeros(3, 4), torch.zeros(3, 2)
    w1, w2 = torch.zeros(16, 4), torch.zeros(4, 8)
    targets, row = torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    for size in (2 ** 31 - 1, 2 ** 31, 2 ** 31 + 512, 3 * 2 ** 31 + 256):
        ws = torch.empty(size, dtype=torch.uint8)  # (never touched, so it takes no memory)
        for call in (lambda: B.layernormBackward(Nowhere, x, x, x, None, stats, workspace=ws),
                     lambda: B.gatedFeedForwardForward(Nowhere, x, w1, w2, x, workspace=ws), lambda: B.gatedFeedForwardBackward(Nowhere, x, w1, w2, x, workspace=ws),
                     lambda: B.softmaxCrossEntropyForward(Nowhere, x, x, targets, row, workspace=ws),
                     lambda: B.softmaxCrossEntropyBackward(Nowhere, x, x, targets, row, workspace=ws)):
            with pytest.raises(B.BackendError, match="null context"):  # everything described, and the library asked
                call()
    with pytest.raises(B.BackendError, match="dense row-major"):
        B.layernormBackward(Nowhere, x, x, x, None, stats, workspace=torch.empty(64, 2, dtype=torch.uint8).T)


@pytest.mark.gpu
def test_all_of_a_large_workspace_counts(ctx):
    """Wide products over many tokens take more than 2 GB of scratch memory; every byte the size function asks for is needed."""
    from minml_b200 import backend as B
    tokens, embed, hidden = 400000, 64, 1024
    x = torch.randn((tokens, embed), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    w1, w2 = torch.randn((2 * hidden, embed), device="cuda").half() / 8, torch.randn((embed, hidden), device="cuda").half() / 32
    size = B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, x.dtype, True, False)
    assert size > 2 ** 31
    ws = torch.empty(size, device="cuda", dtype=torch.uint8)
    dx, dw1, dw2 = torch.empty_like(x), torch.empty_like(w1), torch.empty_like(w2)
    B.gatedFeedForwardBackward(ctx, x, w1, w2, x, dx, dw1, dw2, workspace=ws)
    ctx.synchronize()
    with pytest.raises(B.BackendError, match="are needed"):
        B.gatedFeedForwardBackward(ctx, x, w1, w2, x, dx, dw1, dw2, workspace=ws[:-512])
    few = slice(tokens - 100, tokens)
    want, part = torch.empty_like(dx[few]), torch.empty(B.gatedFeedForwardGetWorkspaceSize(ctx, x[few].shape, w1.shape, x.dtype, True, False), device="cuda", dtype=torch.uint8)
    B.gatedFeedForwardBackward(ctx, x[few].clone(), w1, w2, x[few].clone(), want, workspace=part)
    ctx.synchronize()
    assert float((dx[few].double() - want.double()).norm() / want.double().norm()) <= 2.0 ** -10  # one more or less cut along K, then one rounding each
