"""Readout4 refuses records whose scales are out of their range, wherever they stand, and no others."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)


def records(rt, models, inputs, heads, outputs, group):
    """Records full of bits, their scales 1; and the scales' view [models, inputs, heads * groups]."""
    per = rt.Readout4.record_bytes(models, inputs, heads, outputs, group)
    padded = -(-outputs // 32) * 32
    nb, ng = heads * padded // 2, heads * -(-padded // group)
    rec = np.full((models, inputs, per), 0xFF, np.uint8)
    scales = np.ones((models, inputs, ng), np.float32)
    return rec, nb, scales


def make(rt, rec, nb, scales, heads, outputs, group):
    bits = (scales.view(np.uint32) >> 16).astype(np.uint16)
    r = rec.copy()
    r[:, :, nb:nb + 2 * bits.shape[2]] = bits.view(np.uint8).reshape(*bits.shape[:2], -1)
    return rt.Readout4(torch.from_numpy(r).cuda(), rec.shape[1], heads, outputs, group)


SHAPES = [(1, 1, 1, 1, 32), (2, 33, 3, 77, 64), (1, 700, 7, 480, 32), (3, 65, 2, 1000, 128)]


@pytest.mark.parametrize("models,inputs,heads,outputs,group", SHAPES)
def test_scales_within_their_range(rt, models, inputs, heads, outputs, group):
    rec, nb, s = records(rt, models, inputs, heads, outputs, group)
    flat = s.reshape(-1)
    for k, v in enumerate((0.0, 2.0 ** -110, 2.0 ** 100, -1.5, -2.0 ** 100, -0.0)):
        flat[k % flat.size] = v
        make(rt, rec, nb, s, heads, outputs, group)


@pytest.mark.parametrize("models,inputs,heads,outputs,group", SHAPES)
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 2.0 ** 101, 1.0078125 * 2.0 ** 100, 2.0 ** -111, -2.0 ** -130,
                                 float("-inf")])
def test_scales_out_of_their_range(rt, models, inputs, heads, outputs, group, bad):
    rec, nb, s = records(rt, models, inputs, heads, outputs, group)
    for at in {0, s.size - 1, s.size // 2}:
        t = s.copy()
        t.reshape(-1)[at] = bad
        with pytest.raises(ValueError, match="scales"):
            make(rt, rec, nb, t, heads, outputs, group)


def test_not_checked_while_a_graph_is_captured(rt):
    r = rt.Readout4.quantize(torch.ones((1, 32, 1, 40), device="cuda"))
    x = torch.ones((1, 32), device="cuda")
    r.matvec(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = rt.Readout4(r.records, 32, 1, 40).matvec(x)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, r.matvec(x))
