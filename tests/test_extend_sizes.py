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


@pytest.mark.parametrize("sizes", [
    dict(n=65536), dict(B=4, n=32768), dict(B=4, Hq=32, H=32, n=65536, T=0), dict(n=(1 << 24) - 8), dict(B=8, Hq=64, H=8, n=131072, T=0),
    dict(B=2, Hq=4096, H=512, n=32768), dict(B=1 << 20, Hq=4, n=16, P=8), dict(n=1 << 20, Hq=8, P=4096), dict(B=(1 << 18) - 1, Hq=128, H=128, n=1, P=8),
    dict(B=2, Hq=8, H=8, n=40000, P=1000, bits=2)], ids=str)
def test_documented_sizes_are_taken(sizes):
    assert _call(**sizes) == WORKSPACE


def test_sizes_that_are_refused():
    assert _call(n=1 << 24) == _call(T=1 << 24, n=1) == _call(P=(1 << 24) + 1) == SHAPE     # tokens
    assert _call(B=1 << 16, Hq=64, H=64, n=256) == SHAPE                                     # 2^30 rows
    assert _call(B=1 << 19, Hq=64, H=64, n=1) == _call(B=1 << 18, Hq=128, H=128, n=1, P=8) == SHAPE      # 2^25 sequences and heads


def test_quotients():
    """The multiplication that stands for a division, at its largest operands."""
    import random
    rng = random.Random(1)
    for d in [2, 3, 7, 65535, 65536, 65537, (1 << 31) - 1, *(rng.randrange(2, 1 << rng.randrange(2, 32)) for _ in range(2000))]:
        mul = ((1 << 64) - 1) // d + 1
        lo, hi = mul & 0xFFFFFFFF, mul >> 32
        for x in [0, 1, d - 1, d, (1 << 31) - 1, (1 << 31) - 1 - (1 << 31) % d, *(rng.randrange(1 << 31) for _ in range(20))]:
            assert (x * hi + (x * lo >> 32)) >> 32 == x // d and x * hi + (x * lo >> 32) < 1 << 64
