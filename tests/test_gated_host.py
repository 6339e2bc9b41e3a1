"""What the gated layer's C entry points refuse beside test_gated_norm_host.py's cases; no GPU."""
import ctypes

import pytest

from ksmm_b200 import _lib
from test_gated_norm_host import gated_desc


@pytest.mark.parametrize("change", [dict(saved_bytes=2 * 8 * 8 * 2 - 1), dict(batch=1000, saved_bytes=4096), dict(offset=16)])
def test_backward_of_less_than_was_kept(change):
    """The backward pass reads as much as the forward pass of these sizes keeps, and refuses less."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 17)
    room = (ctypes.addressof(buf) + 255) // 256 * 256
    layouts, grads = (ctypes.c_int32 * 1)(0), (ctypes.c_void_p * 1)(None)
    change = {"saved_bytes": 65536, **change}
    saved = room + change.pop("offset", 0)
    d = gated_desc(saved=saved, layouts=layouts, workspace=room, workspace_bytes=65536, **change)
    before = lib.ksmm_cu_launch_count()
    assert lib.ksmm_cu_gated_backward(ctypes.byref(d), d.input, None, grads, None, None) == _lib.KSMM_ERR_WORKSPACE
    assert b"kept" in lib.ksmm_cu_last_error() and lib.ksmm_cu_launch_count() == before
