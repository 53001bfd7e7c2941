"""How large a launch may be, and calls past it, without a GPU."""
import ctypes as C

import pytest

from xwen_amd import _lib


@pytest.fixture(scope="module")
def fits():
    f = C.CDLL(_lib.LIB_PATH).xs_host_launch_fits
    f.restype, f.argtypes = C.c_bool, [C.c_int64, C.c_int64]
    return f


@pytest.mark.parametrize("threads", [64, 256, 1024])
def test_a_launch_is_bounded_by_its_work_items(fits, threads):
    most = (2**32 - 1) // threads
    assert fits(0, threads) and fits(1, threads) and fits(most, threads)
    assert not fits(most + 1, threads) and not fits(2**31, threads) and not fits(2**50, threads)
