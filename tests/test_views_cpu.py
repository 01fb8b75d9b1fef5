"""What describes a tensor to the library, without a GPU."""
import numpy as np
import pytest

from qlinear import QlError, _lib


@pytest.mark.parametrize("shape", [(2, 3), [2, 3], np.array([2, 3]), (np.int64(2), 3.0), (n for n in (2, 3)), map(int, "23")])
def test_a_shape_is_any_iterable_of_sizes(shape):
    t = _lib.make_tensor(16, _lib.F32, shape)
    assert (t.data, t.dtype, t.rank, list(t.shape)) == (16, _lib.F32, 2, [2, 3, 0, 0, 0, 0, 0, 0])


def test_ranks():
    assert _lib.make_tensor(None, _lib.I8, ()).rank == 0
    assert _lib.make_tensor(None, _lib.I8, range(1, 9)).rank == 8
    with pytest.raises(QlError, match="rank 9 exceeds 8"):
        _lib.make_tensor(None, _lib.I8, range(9))
