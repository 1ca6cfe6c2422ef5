"""Numbers that do not fit an entry point's 32-bit argument are refused; by itself ctypes passes their lower half on, and a batch of
2^32 + 2 images would be answered as one of two (no GPU needed)."""
import ctypes

import pytest

BIG = [2 ** 31, 2 ** 32 + 2, -2 ** 31 - 1, 2 ** 64 + 2]


@pytest.mark.parametrize("big", BIG)
def test_a_size_that_does_not_fit_is_refused(lib_built, big):
    from dfa3d_b200 import _lib
    for at in range(5):
        args = [2, 9000, 64, 4, 2, 1]
        args[at] = big
        with pytest.raises(RuntimeError, match="dfa3d_group_norm_workspace failed .invalid argument.*32 bits"):
            _lib.size("dfa3d_group_norm_workspace", *args)
    with pytest.raises(RuntimeError, match="32 bits"):
        _lib.size("dfa3d_dropout_add_layer_norm_workspace", 4, big)


@pytest.mark.parametrize("big", BIG)
def test_an_argument_that_does_not_fit_is_refused(lib_built, big):
    from dfa3d_b200 import _lib
    calls = _lib.calls
    with pytest.raises(RuntimeError, match="dfa3d_column_sum failed .invalid argument.*32 bits"):
        _lib.call_plain("dfa3d_column_sum", None, 0, big, None, None)
    assert _lib.calls == calls


@pytest.mark.parametrize("wrong", [1.0, "4", None])
def test_what_is_no_integer_is_refused(lib_built, wrong):
    from dfa3d_b200 import _lib
    with pytest.raises(RuntimeError, match="dfa3d_column_sum failed"):
        _lib.call_plain("dfa3d_column_sum", None, 0, wrong, None, None)


def test_what_fits_is_passed_on(lib_built):
    import numpy as np
    from dfa3d_b200 import _lib
    want = _lib.size("dfa3d_group_norm_workspace", 2, 9000, 64, 4, 2, 1)
    assert want == _lib.size("dfa3d_group_norm_workspace", np.int64(2), ctypes.c_int32(9000).value, 64, 4, 2, True)
    with pytest.raises(RuntimeError, match="B and N"):
        _lib.size("dfa3d_group_norm_workspace", -2 ** 31, 9000, 64, 4, 2, 1)
    with pytest.raises(RuntimeError, match="too many"):
        _lib.size("dfa3d_group_norm_workspace", 1, 2 ** 31 - 1, 64, 4, 2, 1)
