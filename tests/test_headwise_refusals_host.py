"""Head-wise calls at the edges of their arguments, without a GPU."""
from numba_cuda_b200 import _lib
from test_headwise_host import _heads, _rotation


def test_positions_are_checked_where_nothing_is_rotated():
    """They tell padding tokens; without a rotation they may be left out."""
    L = _lib.lib()

    def call(**change):
        return L.b2k_norm_rotate(_rotation(rot=0, cos=0, sin=0, **change), _heads(), _heads(), None)

    assert call(pos=4100) == _lib.ERR_ALIGNMENT
    assert call(pb=2) == _lib.ERR_INVALID_ARG
    assert call(rows=-1) == _lib.ERR_INVALID_ARG
    assert call(tokens=0, pos=0, pb=0) == 0
