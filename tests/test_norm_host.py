"""What residual_norm and its C entry points refuse beside test_gated_norm_host.py's cases; no GPU."""
import ctypes

import pytest

from ksmm_b200 import _lib
from test_gated_norm_host import norm_desc


@pytest.mark.parametrize("key", ["post_weight", "post_bias", "grad_post_weight", "grad_post_bias"])
def test_rows_of_a_post_norm_without_one(key):
    """Some of the kernels would apply them and some would not; the Python call refuses them too."""
    lib = _lib.load()
    p = norm_desc().x
    d = norm_desc(y=p, z=p, stats=(p + 15) // 16 * 16, grad_h=p, **{key: p})
    before = lib.ksmm_cu_launch_count()
    for call in (lib.ksmm_cu_norm_forward, lib.ksmm_cu_norm_backward):
        assert call(ctypes.byref(d), None, 0, None) == _lib.KSMM_ERR_BAD_ARGUMENT
        assert b"post_norm" in lib.ksmm_cu_last_error()
    assert lib.ksmm_cu_norm_backward_workspace_bytes(ctypes.byref(d)) == 0
    assert lib.ksmm_cu_launch_count() == before


def test_pattern_values_keep_their_upper_bits():
    """A value of 2^32 + 5 must not reach the library as 5."""
    assert list(_lib.int32_array([1, 2 ** 31 - 1, -1])) == [1, 2 ** 31 - 1, -1]
    for v in (2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1):
        with pytest.raises(ValueError, match="32-bit"):
            _lib.int32_array([1, v, 2, 3])
