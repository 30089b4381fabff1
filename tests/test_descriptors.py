"""The descriptors that backend.py makes, and the shapes it takes: they need no GPU."""
import torch


def test_an_absent_operand_is_described_anew_every_time():
    """A caller may fill in what it was given; later calls must not see it."""
    from minml_b200 import _abi
    from minml_b200 import backend as B
    d = B.desc(None)
    d.data, d.rank, d.dtype = 4096, 1, _abi.DTYPE_FLOAT32
    d.dim[0] = 7
    again = B.desc(None)
    assert again.data is None and again.rank == 0 and again.dtype == _abi.DTYPE_UNKNOWN and list(again.dim) == [0] * 6


def test_shapes_of_any_iterable_of_numbers():
    import numpy as np
    from minml_b200 import backend as B
    for dims in ((2, 3, 5), [2, 3, 5], torch.Size((2, 3, 5)), np.array([2, 3, 5]), np.array([2.0, 3.0, 5.0]), iter((2, 3, 5)), (n for n in (2.0, 3, np.int64(5))), torch.empty(2, 3, 5)):
        s = B.shape_of(dims)
        assert s.rank == 3 and list(s.dim) == [2, 3, 5, 0, 0, 0]
    assert B.shape_of([]).rank == 0
    d = B.desc(torch.empty(2, 3, dtype=torch.float16))
    assert d.rank == 2 and list(d.dim) == [2, 3, 0, 0, 0, 0]
