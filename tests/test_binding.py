"""What the extension module refuses on the host, before any call into the library: it needs no GPU."""
import pytest
import torch


class Nowhere:
    """Stands for a context whose device is where CPU tensors say they are."""
    handle = None
    device_index = -1


def call(x, stats=None, w=None):
    from minml_b200 import backend as B
    B.layernormForwardTraining(Nowhere, x, x, w, None, torch.zeros(3, 2) if stats is None else stats)


def test_refusals():
    from minml_b200 import backend as B
    x = torch.zeros(3, 4)
    with pytest.raises(B.BackendError, match="null context"):  # everything described, and the library asked
        call(x)
    with pytest.raises(B.BackendError, match="strides"):
        call(x.T)
    with pytest.raises(B.BackendError, match="6 dimensions"):
        call(x, w=torch.zeros(1, 1, 1, 1, 1, 1, 4))
    with pytest.raises(B.BackendError):  # an extent beyond a descriptor's 32 bits
        call(torch.empty(0, 2 ** 31))
    with pytest.raises(AttributeError):
        call([1.0, 2.0])

    class Elsewhere(Nowhere):
        device_index = 0
    with pytest.raises(B.BackendError, match="tensor on cpu"):
        B.layernormForwardTraining(Elsewhere, x, x, None, None, x)
    with pytest.raises(TypeError):
        B._binding.layernorm_forward(None, -1, x)
    with pytest.raises(TypeError):
        B.gatedFeedForwardForward(Nowhere, x, x, x, x, beta="half")
    with pytest.raises(B.BackendError, match="unknown gate"):
        B.gatedFeedForwardForward(Nowhere, x, x, x, x, gate="tanh")


def test_a_refused_call_leaves_its_arguments_alone():
    """References are given back on every way out."""
    import sys
    from minml_b200 import backend as B
    x, tall = torch.zeros(3, 4), torch.zeros(4, 3).T
    before = sys.getrefcount(x), sys.getrefcount(tall), sys.getrefcount(torch.float32), sys.getrefcount(B.BackendError)
    for _ in range(50):
        for bad in (x, tall):
            try:
                call(bad)
            except B.BackendError:
                pass
    after = sys.getrefcount(x), sys.getrefcount(tall), sys.getrefcount(torch.float32), sys.getrefcount(B.BackendError)
    assert all(abs(a - b) < 20 for a, b in zip(before, after))
