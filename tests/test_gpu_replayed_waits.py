"""A bounded wait that runs out in a replayed CUDA graph is reported like one in a call: the operators may be captured, and a replay launches nothing
that the host would see."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_replayed_wait_that_runs_out_is_reported():
    """The small kernel of the library's own test waits (with a limit) on a barrier that nothing completes, gives up and writes the status word."""
    from minml_b200 import backend as B
    ctx = B.Context(0)
    x = torch.randn((300, 64), device="cuda").half()
    y, stats = torch.empty_like(x), torch.empty((300, 2), device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=ctx.torch_stream()):
        B.lib.mb200_selftest_bounded_wait(ctx.handle, 2000)
    ctx.synchronize()  # nothing has run yet
    for _ in range(2):
        with torch.cuda.stream(ctx.torch_stream()):
            graph.replay()
        with pytest.raises(B.BackendError, match="gave up on a bounded wait"):
            ctx.synchronize()
        ctx.synchronize()  # reported once
    B.layernormForwardTraining(ctx, x, y, None, None, stats)  # the context is usable
    ctx.synchronize()
    assert bool(torch.isfinite(y).all())
    del graph
    ctx.close()
