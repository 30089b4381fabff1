"""Extents at the ends of a descriptor's 32 bits are refused on the host, before anything is launched: an index that runs past the end of such a row
would come round to a negative one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_refusals(ctx):
    from minml_b200 import _abi
    from minml_b200 import backend as B
    memory = torch.zeros(64, device="cuda", dtype=torch.float16)

    def tensor(*dims, dtype=_abi.DTYPE_FLOAT16):
        d = _abi.mlTensor_t()
        d.data, d.dtype, d.rank = memory.data_ptr(), dtype, len(dims)
        for i, n in enumerate(dims):
            d.dim[i] = n
        return d
    none, most, f32, i32 = _abi.mlTensor_t(), 2 ** 31 - 1, _abi.DTYPE_FLOAT32, _abi.DTYPE_INT32
    lib, h = B.lib, ctx.handle
    huge = tensor(65536, 65536, 65536, 65536, 8)
    calls = [
        (lambda: lib.mb200_layernorm_forward(h, tensor(1, most), none, none, none, tensor(1, most), tensor(1, 2, dtype=f32)), "too long"),
        (lambda: lib.mb200_layernorm_backward(h, tensor(1, most), none, tensor(1, most), none, tensor(1, 2, dtype=f32), 0.0, tensor(1, most), 0.0, none, none, none), "too long"),
        (lambda: lib.mb200_layernorm_forward(h, huge, none, none, none, huge, tensor(1, 2, dtype=f32)), "more elements"),
        (lambda: lib.mb200_gated_feed_forward_forward(h, tensor(20, 8), tensor(most - 1, 8), tensor(8, 2 ** 30 - 1), 0.0, tensor(20, 8), 2, none, none), "too many"),
        (lambda: lib.mb200_gated_feed_forward_forward(h, huge, tensor(16, 8), tensor(8, 8), 0.0, huge, 2, none, none), "more elements"),
        (lambda: lib.mb200_gated_feed_forward_backward(h, tensor(20, most), tensor(4, most), tensor(most, 2), none, tensor(20, most), 0.0, none, 0.0, none, none, 2, none), "too many"),
        (lambda: lib.mb200_softmax_cross_entropy_forward(h, tensor(2, 8), tensor(most, 8), tensor(2, dtype=i32), tensor(2, dtype=f32), none, none), "too many"),
        (lambda: lib.mb200_softmax_cross_entropy_forward(h, tensor(most, 8), tensor(9, 8), tensor(most, dtype=i32), tensor(most, dtype=f32), none, none), "too many"),
        (lambda: lib.mb200_softmax_cross_entropy_backward(h, tensor(2, 8), tensor(most, 8), tensor(2, dtype=i32), tensor(2, dtype=f32), 1.0, none, 0.0, none, 0.0, none, none), "too many")]
    before = B.launch_count()
    for call, text in calls:
        call()
        with pytest.raises(B.BackendError, match=text):
            ctx.check()
    assert B.launch_count() == before
    assert B.layernormBackwardGetWorkspaceSize(ctx, (1, most)) == 0
    assert B.gatedFeedForwardGetWorkspaceSize(ctx, (20, 8), (most - 1, 8)) == 0
    assert B.softmaxCrossEntropyGetWorkspaceSize(ctx, (2, 8), (most, 8)) == 0
