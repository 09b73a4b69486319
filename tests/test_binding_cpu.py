"""What the Python binding takes for an address: None, an integer, or anything with data_ptr()."""
import ctypes as C

import numpy as np
import pytest

import cfk_b200 as cfk


class Held:
    def data_ptr(self):
        return 0x7000


@pytest.mark.parametrize("bad", [3.7, np.float32(0.3), np.array([5.5]), np.array([0x1000]), np.zeros(4), "123", b"4096", [4096], np.int64(64)])
def test_what_is_no_address_is_refused(lib, bad):
    with pytest.raises(AttributeError):
        cfk._ptr(bad)
    with pytest.raises(AttributeError):
        lib.gemm_i8(0x1000, 0x2000, 0x3000, a_scale=0x4000, b_scale=0x5000, bias=bad, m=4, n=64, k=64, out_dtype=cfk.FP16)
    with pytest.raises(AttributeError):
        lib.gemm(bad, 0x2000, 0x3000, dtype=cfk.FP16, m=128, n=128, k=64)


def test_addresses_pass_unchanged():
    class Code(int):
        pass
    assert cfk._ptr(None) is None and cfk._ptr(0x1000) == 0x1000 and cfk._ptr(Code(48)) == 48 and cfk._ptr(Held()) == 0x7000
    a = cfk.GemmI8Args(cfk.FP16, 1, 1, 1, cfk._ptr(Held()))
    assert C.cast(a.a, C.c_void_p).value == 0x7000


def test_an_error_inside_data_ptr_reaches_the_caller():
    class Broken:
        def data_ptr(self):
            raise AttributeError("no storage")
    with pytest.raises(AttributeError, match="no storage"):
        cfk._ptr(Broken())
