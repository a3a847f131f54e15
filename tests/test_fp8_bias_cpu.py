"""`ha_linear_fp8` takes a residual whose rows are all the same one (a bias), and no other stride below a row."""
import ctypes as C

from hashattention import _ops


def test_residual_strides():
    lib = _ops.load_library()
    buf = (C.c_char * 4096)()
    mem = (C.addressof(buf) + 255) // 256 * 256

    def lin(rs):
        return lib.ha_linear_fp8(mem, 256, mem, 2, mem, mem, mem, rs, 0, mem, 32, _ops.HA_BF16, 4, 32, 256, None, 0, None)

    assert lin(1) == lin(31) == lin(-1) == -2
    if lib.ha_device_count() == 0:
        assert lin(0) == lin(32) == -6
