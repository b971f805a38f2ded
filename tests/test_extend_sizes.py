"""What adkv_extend takes and refuses, on the host: every pointer here is a number, and no call gets as far as a launch (those that
are taken lack workspace)."""
import ctypes

import pytest
import torch

from adkv_amd import _lib

ONE, NULL, SHAPE, ALIGN, WORKSPACE = 256, -1, -3, -5, -7


def _call(B=1, Hq=1, H=1, T=8, n=2, P=0, cap=None, k_new=ONE, v_new=ONE, k_strides=None, v_strides=None, nbytes=0, bits=4):
    arr5 = (ctypes.c_void_p * 5)(*[ONE] * 5)
    st = lambda s: None if s is None else (ctypes.c_int64 * 3)(*s)
    pre = None
    if P:
        arr = ctypes.cast(arr5, ctypes.c_void_p)
        pre = ctypes.byref(_lib.Prefix(k_codes=ONE, v_codes=ONE, k_params=arr, v_params=arr, tokens=P, n_super=-(-P // (32 // bits))))
    return _lib.lib().adkv_extend(ONE, st((n * Hq * 128, 128, Hq * 128)), ONE, ONE, k_new, v_new, st(k_strides), st(v_strides), arr5, arr5, None,
                                  None, 1.0, ONE, B, Hq, H, T, n, 128, cap or -(-(T + n) // (32 // bits)), bits, 1, None, None, 0, 0, pre, ONE,
                                  nbytes, None)


@pytest.fixture(autouse=True)
def no_launches():
    # a call that got further than it should would launch kernels on these pointers
    if torch.cuda.is_available():
        pytest.skip("where there is no device")


ENOUGH = 1 << 62


def test_what_is_refused_is_refused_ahead_of_the_launches():
    """With all the workspace there could be: the first launch would fail with the device's error."""
    assert _call(k_new=258, nbytes=ENOUGH) == _call(v_new=258, nbytes=ENOUGH) == ALIGN
    assert _call(k_strides=(256, 256, 127), nbytes=ENOUGH) == _call(v_strides=(-256, 256, 128), nbytes=ENOUGH) == SHAPE
    assert _call(k_strides=(257, 256, 128), nbytes=ENOUGH) == SHAPE
    assert _call(B=1 << 20, Hq=256, H=32, n=1, nbytes=ENOUGH) == SHAPE       # more rows than one launch joins
