"""A read-out's sizes past 32 bits are refused, not cut to their lower half; refusals of htm_q4_check."""
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("k", range(5))
def test_sizes_past_32_bits_refused(rt, k):
    good = [1, 32, 1, 40, 32]
    assert rt.Readout4.record_bytes(*good) == 64
    for far in (2 ** 31, 2 ** 32, -2 ** 33):
        sizes = list(good)
        sizes[k] += far
        with pytest.raises(ValueError):
            rt.Readout4.record_bytes(*sizes)


def test_check_of_records_refused(rt):
    import ctypes
    L, INV = rt._lib.lib(), rt._lib.HTM_E_INVALID
    s, bad = rt._lib.Q4Shape(1, 32, 1, 40, 32), rt._lib.Q4Shape(1, 32, 1, 40, 48)
    p, odd = ctypes.c_void_p(64), ctypes.c_void_p(72)
    for args in ((None, p, p), (ctypes.addressof(bad), p, p), (ctypes.addressof(s), None, p), (ctypes.addressof(s), odd, p),
                 (ctypes.addressof(s), p, None)):
        assert L.htm_q4_check(*args, None) == INV
