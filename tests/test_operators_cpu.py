"""Refusals of the read-out and beam entry points that need no GPU: the C ABI
checks its arguments before any HIP call, Python before the C ABI."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def shape(rt, models=1, inputs=32, heads=1, outputs=40, group=32):
    return rt._lib.Q4Shape(models, inputs, heads, outputs, group)


def ref(s):
    return ctypes.addressof(s)


def test_record_bytes(rt):
    L = rt._lib.lib()
    for (heads, outputs, group), want in {(1, 480, 32): 320, (7, 480, 32): 1920, (1, 1, 128): 64, (1, 33, 64): 64,
                                          (2, 1000, 128): 1088, (64, 5, 32): 1152}.items():
        s = shape(rt, heads=heads, outputs=outputs, group=group)
        assert L.htm_q4_record_bytes(ref(s)) == want
        assert rt.Readout4.record_bytes(1, 32, heads, outputs, group) == want


@pytest.mark.parametrize("bad", [dict(models=0), dict(inputs=0), dict(inputs=65537), dict(heads=0), dict(heads=65),
                                 dict(outputs=0), dict(outputs=65537), dict(group=16), dict(group=48),
                                 dict(heads=64, outputs=16385)])
def test_shapes_refused(rt, bad):
    L = rt._lib.lib()
    s = shape(rt, **bad)
    assert L.htm_q4_record_bytes(ref(s)) == 0 and L.htm_last_error()
    p = ctypes.c_void_p(64)
    INV = rt._lib.HTM_E_INVALID
    assert L.htm_q4_logits(ref(s), p, p, 1, 1, p, None) == INV
    assert L.htm_q4_probabilities(ref(s), p, p, 1, None, 1, p, None) == INV
    assert L.htm_q4_matvec(ref(s), p, p, 0, 40, 1, p, None, 0, None) == INV
    assert L.htm_q4_quantise(ref(s), p, 0, 1, 1, 1, p, p, None) == INV


def test_read_out_arguments_refused(rt):
    L = rt._lib.lib()
    INV = rt._lib.HTM_E_INVALID
    s, odd, two, wide = shape(rt), shape(rt, inputs=33), shape(rt, models=2), shape(rt, outputs=1025)
    p, q = ctypes.c_void_p(64), ctypes.c_void_p(72)
    assert L.htm_q4_logits(None, p, p, 1, 1, p, None) == INV
    for args in ((ref(s), None, p, 1, 1, p), (ref(s), q, p, 1, 1, p), (ref(s), p, None, 1, 1, p), (ref(s), p, p, 1, 1, None),
                 (ref(s), p, p, 0, 2, p), (ref(s), p, p, 1, -1, p), (ref(s), p, p, 1, 65535 * 32 + 1, p), (ref(odd), p, p, 2, 1, p), (ref(two), p, p, 1, 3, p)):
        assert L.htm_q4_logits(*args, None) == INV
    assert L.htm_q4_logits(ref(s), None, None, 1, 0, None, None) == 0      # no rows: nothing to do
    assert L.htm_q4_probabilities(ref(wide), p, p, 1, None, 1, p, None) == INV
    for args in ((ref(s), p, p, 1, 32, 1, p), (ref(s), p, p, 9, 32, 1, p), (ref(s), p, p, 0, 31, 2, p), (ref(s), p, None, 0, 32, 1, p),
                 (ref(s), p, p, 0, 32, 1, None), (ref(two), p, p, 0, 32, 1, p)):
        assert L.htm_q4_matvec(*args, None, 0, None) == INV
    for args in ((None, 0, 1, 1, 1, p, p), (p, 2, 1, 1, 1, p, p), (p, 0, -1, 1, 1, p, p), (p, 0, 1, 1, 1, q, p), (p, 0, 1, 1, 1, p, None)):
        assert L.htm_q4_quantise(ref(s), *args, None) == INV
    assert L.htm_cls_quantise(None, 0, 0, ref(s), p, p, p, None) == INV


def test_beam_arguments_refused(rt):
    L = rt._lib.lib()
    INV = rt._lib.HTM_E_INVALID
    p = ctypes.c_void_p(64)

    def select(groups=1, win=2, wout=2, v=8, dtype=0, x=p, score=p, o=p, gs=16, bs=8):
        return L.htm_beam_select(x, dtype, gs, bs, score, None, groups, win, wout, v, o, o, o, None, 0, None)

    for bad in (dict(groups=-1), dict(win=0), dict(win=65), dict(wout=0), dict(wout=65), dict(v=0), dict(win=64, v=2 ** 25),
                dict(dtype=1), dict(dtype=7), dict(x=None), dict(score=None), dict(o=None), dict(gs=-1), dict(bs=-1)):
        assert select(**bad) == INV, bad
    assert select(groups=0, x=None) == 0
    one = lambda *a: (ctypes.c_void_p * len(a))(*a)  # noqa: E731
    size = lambda *a: (ctypes.c_size_t * len(a))(*a)  # noqa: E731

    def reorder(n=1, src=one(4096), dst=one(8192), b=size(16), parent=ctypes.c_void_p(64), groups=2, beams=4):
        return L.htm_beam_reorder(n, src, dst, b, parent, groups, beams, None)

    for bad in (dict(n=0), dict(n=33), dict(src=None), dict(dst=None), dict(b=None), dict(groups=-1), dict(beams=0),
                dict(beams=65), dict(parent=None), dict(src=one(None)), dict(dst=one(None)), dict(b=size(1 << 40)),
                dict(dst=one(4096 + 64)), dict(dst=one(32)),                          # its source, the parents
                dict(n=2, src=one(4096, 4096), dst=one(8192, 8192 + 127), b=size(16, 16)),
                dict(n=2, src=one(4096, 8192), dst=one(8192, 16384), b=size(16, 16))):  # read here, written there
        assert reorder(**bad) == INV, bad
    assert reorder(groups=0) == 0
    assert L.htm_reorder_streams(None, p, 2, None) == INV
    assert L.htm_copy_streams(None, None, p, None) == INV


def test_scratch_refused(rt):
    """Too little scratch, none, or at an odd address, wherever a call needs some."""
    L = rt._lib.lib()
    INV = rt._lib.HTM_E_INVALID
    p = ctypes.c_void_p(4096)
    for rows, dtype in ((1, 0), (2, 2), (4, 3), (16, 0)):
        s = shape(rt, inputs=24576, heads=1, outputs=480)
        need = L.htm_q4_work_bytes(ref(s), rows)
        assert need and need % (4 * rows * 480) == 0
        for work, nb in ((None, need), (p, need - 1), (p, 0), (ctypes.c_void_p(4098), need)):
            assert L.htm_q4_matvec(ref(s), p, p, dtype, 24576, rows, p, work, nb, None) == INV
    assert L.htm_q4_work_bytes(ref(shape(rt)), 0) == 0 and L.htm_q4_work_bytes(None, 1) == 0
    for win, wout, v in ((1, 1, 8193), (64, 64, 1000), (8, 8, 1 << 20)):
        need = L.htm_beam_work_bytes(3, win, wout, v)
        assert need >= 3 * win * wout * 8
        for work, nb in ((None, need), (p, need - 1), (p, 0), (ctypes.c_void_p(4100), need)):
            assert L.htm_beam_select(p, 0, win * v, v, p, None, 3, win, wout, v, p, p, p, work, nb, None) == INV
    assert L.htm_beam_work_bytes(3, 8, 8, 480) == 0 and L.htm_beam_work_bytes(0, 8, 8, 1 << 20) == 0


def test_tensors_off_the_gpu_refused(rt):
    with pytest.raises(ValueError):
        rt.Readout4(torch.zeros((1, 32, 64), dtype=torch.uint8), 32, 1, 40)
    with pytest.raises(ValueError):
        rt.Readout4.quantize(torch.zeros((1, 32, 1, 40)))
    with pytest.raises(ValueError):
        rt.beam_select(torch.zeros((1, 2, 8)), torch.zeros((1, 2)), 2)
    with pytest.raises(ValueError):
        rt.beam_select(torch.zeros((1, 2, 8), dtype=torch.int32), torch.zeros((1, 2)), 2)
    with pytest.raises(ValueError):
        rt.beam_reorder([torch.zeros((2, 4))], torch.zeros((1, 2), dtype=torch.int32))
