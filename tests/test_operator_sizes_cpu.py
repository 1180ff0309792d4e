"""A read-out's sizes past 32 bits are refused, not cut to their lower half."""
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
