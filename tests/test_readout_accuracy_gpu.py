"""Readout4 where weights of very different size meet: the results keep the bound that float32 sums of exact weights have.

A weight s * (c - 8) has at most 11 significant bits and is exact in float32.  A sum of n of them rounds at most n times,
in whatever order, so |y - y64| <= (n + 2) * 2^-24 * sum |x w| per output: a weight of zero adds nothing, however large
its scale."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

EPS = 2.0 ** -24


def spread(rt, models, inputs, heads, outputs, group, decades, seed):
    """Scales over `decades` powers of ten, and no weight but zero under most of the larger ones."""
    rng = np.random.default_rng(seed)
    padded = -(-outputs // 32) * 32
    groups = -(-padded // group)
    per = rt.Readout4.record_bytes(models, inputs, heads, outputs, group)
    s = 10.0 ** rng.uniform(-decades / 2, decades / 2, (models, inputs, heads, groups))
    code = rng.integers(0, 16, (models, inputs, heads, padded))
    zero = np.repeat(s, group, -1)[..., :padded] > 10.0 ** (-decades / 4)
    code[zero & (rng.random(code.shape) < 0.97)] = 8
    bits = (s.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)
    nb = heads * padded // 2
    rec = np.zeros((models, inputs, per), np.uint8)
    flat = code.reshape(models, inputs, -1).astype(np.uint8)
    rec[:, :, :nb] = flat[..., 0::2] | flat[..., 1::2] << 4
    rec[:, :, nb:nb + 2 * heads * groups] = bits.reshape(models, inputs, -1).view(np.uint8)
    s = (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    w = ((code - 8.0) * np.repeat(s, group, -1)[..., :padded])[..., :outputs]
    return rt.Readout4(torch.from_numpy(rec).cuda(), inputs, heads, outputs, group), w


def words(dense):
    b = np.packbits(dense.astype(np.uint8), axis=1, bitorder="little")
    return torch.from_numpy(np.ascontiguousarray(b).view(np.int32).copy()).cuda()


SHAPES = [  # rows, models, inputs, heads, outputs, group, filled
    (1, 1, 2048, 1, 480, 32, 0.4), (3, 1, 4096, 2, 480, 64, 0.3), (70, 1, 2048, 1, 1000, 128, 0.2),
    (4, 2, 1024, 7, 33, 32, 0.5), (300, 3, 512, 1, 40, 32, 0.9), (2, 2, 3136, 3, 512, 32, 0.3),
]


@pytest.mark.parametrize("decades", [2, 5, 9])
@pytest.mark.parametrize("rows,models,inputs,heads,outputs,group,filled", SHAPES)
def test_scales_of_very_different_size(rt, rows, models, inputs, heads, outputs, group, filled, decades):
    r, w = spread(rt, models, inputs, heads, outputs, group, decades, rows + outputs)
    x = np.random.default_rng(decades).random((rows, inputs)) < filled
    got = r.logits(words(x)).cpu().numpy().astype(np.float64)
    p = r.probabilities(words(x)).cpu().numpy().astype(np.float64)
    v = r.matvec(torch.from_numpy(x).float().cuda()).cpu().numpy().astype(np.float64)
    for k in range(rows):
        m = w[k // (rows // models)][x[k]]
        y, tol = m.sum(0), (len(m) + 2) * EPS * np.abs(m).sum(0)
        assert np.all(np.abs(got[k] - y) <= tol), float((np.abs(got[k] - y) - tol).max())
        # (five and more rows of numbers: up to six exact parts a weight, of one sign)
        assert np.all(np.abs(v[k] - y) <= (tol if rows // models < 5 else 6 * tol))
        e = np.exp(y - y.max(-1, keepdims=True))
        q, d = e / e.sum(-1, keepdims=True), tol.max(-1, keepdims=True)
        # (below float32's normal numbers expf is off by up to a step of 2^-149, the division by half of one)
        assert np.all(np.abs(p[k] - q) <= q * (np.expm1(2 * d) + (outputs + 12) * EPS) + 2 * 2.0 ** -149)


def test_a_weight_of_zero_under_a_large_scale(rt):
    """All active inputs but two have the code of zero: the sums are exact, whatever the order."""
    n = 640
    rec = np.full((1, n, 64), 0x88, np.uint8)                   # 40 outputs, group 32: 32 bytes of codes, two scales
    scale = np.full((n, 2), 2.0 ** 16, np.float32)
    for i, code in ((37, 9), (611, 11)):
        rec[0, i, :32] = code * 0x11
        scale[i] = 2.0 ** -10
    rec[0, :, 32:36] = (scale.view(np.uint32) >> 16).astype(np.uint16).view(np.uint8)
    r = rt.Readout4(torch.from_numpy(rec).cuda(), n, 1, 40)
    y = r.logits(words(np.ones((3, n), bool)))
    assert torch.all(y == 4 * 2.0 ** -10)


def uniform(rt, n, codes, scale):
    """[1, n, 1, 40] with one scale and `codes` [n]."""
    rec = np.zeros((1, n, 64), np.uint8)
    rec[0, :, :32] = (np.asarray(codes) * 0x11)[:, None]
    rec[0, :, 32:36] = (np.full((n, 2), scale, np.float32).view(np.uint32) >> 16).astype(np.uint16).view(np.uint8)
    return rt.Readout4(torch.from_numpy(rec).cuda(), n, 1, 40)


@pytest.mark.parametrize("rows", [1, 2, 4, 6])
def test_large_finite_numbers_meet_zero_weights(rt, rows):
    """scale * x would overflow where x * (scale * (code - 8)) does not: a zero weight adds nothing to a finite x."""
    n = 70
    codes = np.full(n, 8)
    codes[[3, 64]] = 9, 7
    r = uniform(rt, n, codes, 8.0)
    x = torch.full((rows, n), 1e38, device="cuda")
    x[:, 3], x[:, 64] = 3.0, 5.0
    assert torch.all(r.matvec(x) == 8.0 * 3 - 8.0 * 5)
    x[:, 10] = -3e38
    assert torch.all(r.matvec(x) == 8.0 * 3 - 8.0 * 5)


@pytest.mark.parametrize("rows", [1, 2, 4])
def test_small_numbers_keep_their_weights(rt, rows):
    """scale * x lies below float32's numbers, x * (scale * (code - 8)) does not: 2^-151 * 6 = 1.5 * 2^-149 rounds to
    2 * 2^-149, not to 0 (one term, so that nothing is rounded twice)."""
    r = uniform(rt, 33, np.full(33, 14), 2.0 ** -31)
    x = torch.zeros((rows, 33), device="cuda")
    x[:, 32] = 2.0 ** -120
    assert torch.all(r.matvec(x) == 2 * 2.0 ** -149)
