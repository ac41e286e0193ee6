"""Host-side checks of the channel operators' calls that need no GPU: what is refused before anything is launched."""
import ctypes

from deltacnn_b200 import _lib
from deltacnn_b200._lib import lib


def test_first_frame_of_the_delta_norm_refuses_bad_arguments():
    buf = (ctypes.c_uint8 * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256                      # never dereferenced: every call is refused first
    null, unsupported, shape, dtype = 1, 2, 4, 5
    f32, f16, bf16 = _lib.DC_F32, _lib.DC_F16, _lib.DC_BF16
    first = lib.dc_layer_norm_delta_first
    assert first(None, p, p, p, 1, 8, f32, f32, 1e-5, None) == null
    assert first(p, p, p, None, 1, 8, f32, f32, 1e-5, None) == null
    assert first(p, p, p, p, -1, 8, f32, f32, 1e-5, None) == shape
    assert first(p, p, p, p, 1, 0, f32, f32, 1e-5, None) == shape
    assert first(p, p, p, p, 1, (1 << 30) + 1, f32, f32, 1e-5, None) == shape
    assert first(p, p, p, p, 1, 8, bf16, bf16, 1e-5, None) == dtype
    assert first(p, p, p, p, 1, 8, f32, f16, 1e-5, None) == dtype
    assert first(p, p, p, p, 1, 9001, f32, f32, 1e-5, None) == unsupported
    assert first(p, p, p, p, 0, 8, f32, f32, 1e-5, None) == 0
