"""Readout4 (csrc/readout.hip): 4-bit matrix-vector products with group scales
against float64 sums of the same weights.

Tolerance: a weight s * (c - 8) is exact in float32 (8 + 4 bits); a product
with x rounds once and a sum of n terms n times at most, in whatever order, so
|y - y64| <= (n + 2) * 2^-24 * sum |x w| per output.  matvec of five and more rows
a matrix adds up to six exact products a weight instead, all of one sign, so that
their absolute values sum to |x w|: what can be proved for any order is 6 n in
place of n.  logits and
probabilities sum s * c and take 8 * sum s off at the end: what can be proved
has sum s (c + 8) in place of sum |x w|.  All are held to the first bound here,
since so many roundings do not all fall to one side.  softmax: an error d of
the logits moves a probability by a factor within exp(+-2 d), expf and the
division round to 3 * 2^-23 and the sum of k terms to k * 2^-24."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

EPS = 2.0 ** -24


def up(n, to):
    return -(-n // to) * to


def make(rt, models, inputs, heads, outputs, group, seed=0, size=1.0):
    """A read-out of random codes and scales, and its float64 weights [models, inputs, heads, outputs]."""
    rng = np.random.default_rng(seed)
    padded = up(outputs, 32)
    groups = -(-padded // group)
    per = rt.Readout4.record_bytes(models, inputs, heads, outputs, group)
    rec = rng.integers(0, 256, (models, inputs, per), dtype=np.uint8)
    s32 = ((rng.random((models, inputs, heads, groups)) * 0.1 + 0.001) * size).astype(np.float32)
    bits = (s32.view(np.uint32) >> 16).astype(np.uint16)
    nb = heads * padded // 2
    rec[:, :, nb:nb + 2 * heads * groups] = bits.reshape(models, inputs, -1).view(np.uint8)
    q = np.stack((rec[:, :, :nb] & 15, rec[:, :, :nb] >> 4), -1).reshape(models, inputs, heads, padded).astype(np.float64) - 8
    s = (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    w = (q * np.repeat(s, group, -1)[..., :padded])[..., :outputs]
    r = rt.Readout4(torch.from_numpy(rec).cuda(), inputs, heads, outputs, group)
    return r, w


def words(dense):
    b = np.packbits(dense.astype(np.uint8), axis=1, bitorder="little")
    return torch.from_numpy(np.ascontiguousarray(b).view(np.int32).copy()).cuda()


def expect(w, x):
    """float64 y and its bound, x [rows, inputs]."""
    per = x.shape[0] // w.shape[0]
    y = np.zeros((x.shape[0],) + w.shape[2:])
    tol = np.zeros_like(y)
    for r in range(x.shape[0]):
        m = w[r // per]
        i = np.nonzero(x[r])[0]
        y[r] = np.tensordot(x[r, i], m[i], 1)
        tol[r] = (len(i) + 2) * EPS * np.tensordot(np.abs(x[r, i]), np.abs(m[i]), 1)
    return y, tol


def near(got, y, tol):
    d = np.abs(got.cpu().numpy().astype(np.float64) - y)
    assert np.all(d <= tol), (float((d - tol).max()), np.unravel_index((d - tol).argmax(), d.shape))


SHAPES = [  # rows, models, inputs, heads, outputs, group
    (1, 1, 32, 1, 1, 32), (3, 1, 64, 1, 31, 32), (2, 2, 96, 3, 33, 64), (5, 1, 2048, 1, 480, 128),
    (4, 2, 1024, 7, 480, 32), (1, 1, 24576, 7, 480, 32), (6, 3, 320, 2, 1000, 128), (1, 1, 65536, 1, 100, 64),
    (300, 1, 768, 1, 479, 32), (2, 1, 128, 1, 4099, 64), (7, 7, 128, 64, 5, 32), (16, 2, 8192, 1, 1024, 64),
]


@pytest.mark.parametrize("rows,models,inputs,heads,outputs,group", SHAPES)
@pytest.mark.parametrize("filled", [0.01, 0.3])
def test_logits(rt, rows, models, inputs, heads, outputs, group, filled):
    if filled > 0.1 and models * inputs * heads * outputs > 5e7:
        filled = 0.05
    r, w = make(rt, models, inputs, heads, outputs, group)
    rng = np.random.default_rng(1)
    x = rng.random((rows, inputs)) < filled
    got = r.logits(words(x))
    assert got.shape == (rows, heads, outputs) and got.dtype == torch.float32
    near(got, *expect(w, x.astype(np.float64)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,models,inputs,heads,outputs,group", SHAPES + [(1, 1, 1, 1, 1, 32), (9, 1, 37, 1, 480, 32),
                                                                               (17, 1, 4097, 2, 65, 128), (6, 2, 33, 1, 7, 64)])
def test_matvec(rt, rows, models, inputs, heads, outputs, group, dtype):
    r, w = make(rt, models, inputs, heads, outputs, group)
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((rows, inputs))).to(dtype)
    x[:, rng.random(inputs) < 0.3] = 0
    got = r.matvec(x.cuda())
    near(got, *expect(w, x.double().numpy()))


@pytest.mark.parametrize("rows,models,inputs,heads,outputs,group", [(3, 1, 64, 1, 31, 32), (4, 2, 1024, 7, 480, 32),
                                                                    (6, 3, 320, 2, 1000, 128), (2, 1, 128, 1, 1024, 64),
                                                                    (65, 1, 640, 1, 480, 64), (1, 1, 32, 1, 1, 32)])
def test_probabilities(rt, rows, models, inputs, heads, outputs, group):
    r, w = make(rt, models, inputs, heads, outputs, group)
    rng = np.random.default_rng(3)
    x = rng.random((rows, inputs)) < 0.05
    y, tol = expect(w, x.astype(np.float64))
    for live in (None, np.full(models, outputs), rng.integers(1, outputs + 1, models), np.full(models, 1)):
        lv = None if live is None else torch.tensor(live, dtype=torch.int32, device="cuda")
        got = r.probabilities(words(x), lv).cpu().numpy().astype(np.float64)
        for k in range(rows):
            n = outputs if live is None else int(live[k // (rows // models)])
            e = np.exp(y[k, :, :n] - y[k, :, :n].max(-1, keepdims=True))
            p = e / e.sum(-1, keepdims=True)
            d = tol[k, :, :n].max(-1, keepdims=True)
            assert np.all(np.abs(got[k, :, :n] - p) <= p * (np.expm1(2 * d) + 6 * EPS + (n + 6) * EPS) + 1e-45)
            assert np.all(got[k, :, n:] == 0)


def test_probabilities_live_out_of_range(rt):
    """live 0 and below: no bucket is in use, all zero; above n_outputs: all of them."""
    r, _ = make(rt, 3, 64, 1, 40, 32)
    x = words(np.random.default_rng(4).random((3, 64)) < 0.2)
    got = r.probabilities(x, torch.tensor([0, -5, 1000], dtype=torch.int32, device="cuda"))
    assert torch.all(got[:2] == 0)
    assert torch.equal(got[2], r.probabilities(x)[2])


def test_empty_and_full_patterns(rt):
    r, w = make(rt, 1, 4096, 2, 100, 32)
    x = np.zeros((4, 4096), bool)
    x[1, 4095] = x[2, 0] = True
    x[3] = True
    got = r.logits(words(x))
    near(got, *expect(w, x.astype(np.float64)))
    assert torch.all(got[0] == 0)
    assert r.logits(words(x)[:0]).shape == (0, 2, 100)
    assert r.matvec(torch.zeros((0, 4096), device="cuda")).shape == (0, 2, 100)
    # nothing learned yet: every bucket in use is as likely
    p = r.probabilities(words(x))[0]
    assert torch.allclose(p, torch.full_like(p, 0.01), rtol=4 * 2.0 ** -23, atol=0)


def test_strides_offsets_and_out(rt):
    r, w = make(rt, 1, 2048, 1, 480, 32)
    rng = np.random.default_rng(5)
    x = rng.random((6, 2048)) < 0.05
    p = words(x)
    wide = torch.full((6, 100), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:67] = p
    want = r.logits(p)
    assert torch.equal(r.logits(wide[:, 3:67]), want)
    assert torch.equal(r.logits(p.view(torch.uint32)), want)
    assert torch.equal(r.logits(p[::2]), want[::2])
    assert torch.equal(r.logits(p[:1].expand(6, 64)), want[:1].expand(6, 1, 480))
    assert torch.equal(r.logits(p.t().contiguous().t()), want)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        v = torch.from_numpy(rng.standard_normal((6, 2048))).to(dtype).cuda()
        want = r.matvec(v)
        odd = torch.zeros((6, 2051), dtype=dtype, device="cuda")
        odd[:, 1:2049] = v
        assert torch.equal(r.matvec(odd[:, 1:2049]), want)
        guard = torch.full((8, 1, 480), 7.0, device="cuda")
        out = guard[1:7]
        assert r.matvec(v, out=out) is out
        assert torch.equal(out, want) and torch.all(guard[0] == 7) and torch.all(guard[7] == 7)


def test_infinite_and_nan_inputs_stay_in_their_row(rt):
    r, w = make(rt, 1, 256, 1, 64, 32)
    x = torch.from_numpy(np.random.default_rng(6).standard_normal((5, 256))).float().cuda()
    want = r.matvec(x)
    bad = x.clone()
    bad[1, 3], bad[3, 200] = float("nan"), float("inf")
    got = r.matvec(bad)
    assert torch.equal(got[[0, 2, 4]], want[[0, 2, 4]])
    assert torch.all(got[1].isnan()) and not torch.any(got[3].isfinite() & torch.from_numpy(w[0, 200, :, :] != 0).cuda())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 20])
def test_an_infinite_input_by_the_formula(rt, rows, dtype):
    """inf * w is an infinity of w's sign, NaN where w is zero, whatever the bits of the scales."""
    r, w = make(rt, 1, 300, 2, 77, 64)
    x = torch.from_numpy(np.random.default_rng(10).standard_normal((rows, 300))).to(dtype).cuda()
    x[rows - 1, 290], x[0, 7] = float("-inf"), float("inf")
    got = r.matvec(x).cpu().numpy()
    with np.errstate(invalid="ignore"):
        for row, k in ((rows - 1, 290), (0, 7)) if rows > 1 else ():
            assert np.array_equal(got[row], float(x[row, k]) * w[0, k], equal_nan=True)
        if rows == 1:
            assert np.array_equal(got[0], np.inf * w[0, 7] - np.inf * w[0, 290], equal_nan=True)


@pytest.mark.parametrize("size", [2.0 ** -122, 2.0 ** -100, 2.0 ** 100])
@pytest.mark.parametrize("rows", [1, 3, 6, 17])
def test_small_and_large_numbers(rt, rows, size):
    """The same bound far from 1; below float32's normal numbers 2^-149 more a product (each of the six exact ones).
    Five and more rows go through matrix instructions, which take an operand or a result below 2^-126 as zero: of a
    number's three parts that loses less than 3 * 2^-126 times the weight, of the six products and of the six sums
    less than 2^-126 each."""
    r, w = make(rt, 1, 700, 1, 96, 32)
    x = torch.from_numpy(np.random.default_rng(11).standard_normal((rows, 700)) * size).float()
    y, tol = expect(w, x.double().numpy())
    lost = (12 + 3 * np.abs(w).max()) * 700 * 2.0 ** -126 if rows >= 5 else 6 * 700 * 2.0 ** -149
    near(r.matvec(x.cuda()), y, tol + lost)


@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** 103])
@pytest.mark.parametrize("rows", [1, 3, 6])
def test_small_and_large_scales(rt, rows, size):
    """Scales next to both ends of their range, 2^-110 .. 2^100."""
    r, w = make(rt, 1, 700, 1, 96, 32, size=size)
    x = torch.from_numpy(np.random.default_rng(15).standard_normal((rows, 700)) / size).float()
    near(r.matvec(x.cuda()), *expect(w, x.double().numpy()))
    p = np.random.default_rng(16).random((rows, 704)) < 0.1
    r, w = make(rt, 1, 704, 1, 96, 32, size=size)
    near(r.logits(words(p)), *expect(w, p.astype(np.float64)))


@pytest.mark.parametrize("rows,models", [(36, 2), (66000, 66000), (66000, 1), (140000, 7)])
def test_matvec_of_many_rows(rt, rows, models):
    """Passes behind the first, and more rows than one grid dimension holds, for both kernels."""
    r, w = make(rt, models, 64, 1, 40, 32)
    x = torch.from_numpy(np.random.default_rng(12).standard_normal((rows, 64))).float()
    got = r.matvec(x.cuda()).cpu().numpy().astype(np.float64)
    f = x.double().numpy().reshape(models, rows // models, 64)
    y = (f @ w[:, :, 0]).reshape(rows, 1, 40)
    tol = (np.abs(f) @ np.abs(w[:, :, 0])).reshape(rows, 1, 40) * (64 + 2) * EPS
    assert np.all(np.abs(got - y) <= tol)


@pytest.mark.parametrize("rows,models", [(66000, 66000), (66000, 1)])
def test_logits_of_many_rows(rt, rows, models):
    r, w = make(rt, models, 64, 1, 40, 32)
    x = np.random.default_rng(13).random((rows, 64)) < 0.2
    got = r.logits(words(x)).cpu().numpy().astype(np.float64)
    f = x.astype(np.float64).reshape(models, rows // models, 64)
    y = (f @ w[:, :, 0]).reshape(rows, 1, 40)
    tol = (f @ np.abs(w[:, :, 0])).reshape(rows, 1, 40) * (64 + 2) * EPS
    assert np.all(np.abs(got - y) <= tol)
    p = r.probabilities(words(x)).cpu().numpy()
    assert np.all(np.abs(p.sum(-1) - 1) <= 1e-5) and np.array_equal(p.argmax(-1), got.argmax(-1))


def test_records_past_32_bits(rt):
    """The last models of 5.2 GB of records: offsets of more than 32 bits."""
    ni, no, nm = 16384, 480, 1170
    per = rt.Readout4.record_bytes(nm, ni, 1, no)
    rec = torch.zeros((nm, ni, per), dtype=torch.uint8, device="cuda")
    assert rec.numel() > 2 ** 32
    one, w = make(rt, 2, ni, 1, no, 32)
    assert one.records.shape[2] == per
    rec[-2:] = one.records
    r = rt.Readout4(rec, ni, 1, no)
    rng = np.random.default_rng(14)
    x = rng.random((nm, ni)) < 0.01
    got = r.logits(words(x))
    assert torch.all(got[:-2] == 0)
    assert torch.equal(got[-2:], one.logits(words(x[-2:])))
    near(got[-2:], *expect(w, x[-2:].astype(np.float64)))
    for rows in (1, 5):
        v = torch.from_numpy(rng.standard_normal((nm * rows, ni)).astype(np.float32) * (rng.random(ni) < 0.05)).float()
        near(r.matvec(v.cuda())[-2 * rows:], *expect(w, v[-2 * rows:].double().numpy()))


def test_deterministic_and_on_another_stream(rt):
    r, _ = make(rt, 1, 24576, 7, 480, 32)
    rng = np.random.default_rng(7)
    p = words(rng.random((9, 24576)) < 0.02)
    x = torch.from_numpy(rng.standard_normal((9, 24576))).float().cuda()
    a, b = r.logits(p), r.matvec(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append((r.logits(p), r.matvec(x)))
    torch.cuda.synchronize()
    for c, d in outs:
        assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.parametrize("rows", [1, 4, 6])
def test_captured_into_graphs(rt, rows):
    """Two graphs of the same read-out, replayed in turn with eager calls between, give the eager results."""
    r, _ = make(rt, 1, 24576, 1, 480, 32)
    rng = np.random.default_rng(8)
    p = words(rng.random((rows, 24576)) < 0.02)
    x = torch.from_numpy(rng.standard_normal((rows, 24576))).to(torch.bfloat16).cuda()
    graphs = []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        r.logits(p), r.probabilities(p), r.matvec(x)
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = (r.logits(p), r.probabilities(p), r.matvec(x))
        graphs.append((g, outs))
    for k in range(6):
        p.copy_(words(rng.random((rows, 24576)) < 0.02))
        x.copy_(torch.from_numpy(rng.standard_normal((rows, 24576))))
        g, outs = graphs[k % 2]
        g.replay()
        want = (r.logits(p), r.probabilities(p), r.matvec(x))
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_quantize(rt, group, dtype):
    """Codes and scales as defined, zeros exactly zero, any strides of the first three dimensions."""
    rng = np.random.default_rng(9)
    w = torch.from_numpy(rng.standard_normal((2, 40, 3, 77)) * 10.0 ** rng.integers(-30, 6, (2, 40, 3, 1))).to(dtype)
    w[0, 3] = 0
    w[1, 5, 1, 20:] = 0
    w[rng.random(w.shape) < 0.3] = 0
    r = rt.Readout4.quantize(w.cuda(), group)
    rec = r.records.cpu().numpy()
    padded, groups = 96, -(-96 // group)
    nb = 3 * padded // 2
    q = np.stack((rec[:, :, :nb] & 15, rec[:, :, :nb] >> 4), -1).reshape(2, 40, 3, padded).astype(np.int64) - 8
    s = rec[:, :, nb:nb + 6 * groups].copy().view(np.uint16).reshape(2, 40, 3, groups)
    f = w.double().numpy()
    for g in range(groups):
        part = np.zeros((2, 40, 3, min(group, padded - g * group)))
        live = f[..., g * group:(g + 1) * group]
        part[..., :live.shape[-1]] = live
        want = torch.from_numpy(np.abs(part).max(-1) / 7).float().to(torch.bfloat16)
        assert np.array_equal(s[..., g], want.view(torch.int16).numpy().view(np.uint16))
        sc = want.double().numpy()[..., None]
        with np.errstate(divide="ignore", invalid="ignore"):
            code = np.where(sc > 0, np.clip(np.rint(part / sc), -7, 7), 0)
        assert np.array_equal(q[..., g * group:g * group + part.shape[-1]], code)
    # the same matrix through transposed storage
    t = w.cuda().permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)
    assert not t.is_contiguous() and torch.equal(rt.Readout4.quantize(t, group).records, r.records)
    # half a step of the group's scale (rounded to bfloat16: 1 + 2^-8) is the most a weight is off
    y = np.zeros((2, 40, 3, 77))
    for i in range(40):
        x = torch.zeros((2, 40), device="cuda")
        x[:, i] = 1
        y[:, i] = r.matvec(x).cpu().numpy()
    step = np.repeat((s.astype(np.uint32) << 16).view(np.float32).astype(np.float64), group, -1)[..., :77]
    assert np.all(np.abs(y - f) <= step * 0.5 * (1 + 2.0 ** -6) + 1e-37)


def test_quantize_refuses_nonfinite(rt):
    w = torch.zeros((1, 8, 1, 40), device="cuda")
    for v in (float("inf"), float("nan")):
        w[0, 5, 0, 39] = v
        with pytest.raises(ValueError, match="finite"):
            rt.Readout4.quantize(w)


def test_quantize_below_its_range(rt):
    """A group whose scale would lie below 2^-110 is zero; the next one at 2^-110 is not."""
    w = torch.zeros((1, 4, 1, 64), device="cuda", dtype=torch.float64)
    w[0, 1, 0, :32], w[0, 1, 0, 32:] = 6.99 * 2.0 ** -110, 7 * 2.0 ** -110
    y = rt.Readout4.quantize(w).matvec(torch.full((1, 4), 2.0 ** 60, device="cuda"))[0, 0]
    assert torch.all(y[:32] == 0) and torch.all(y[32:] == 7 * 2.0 ** -50)


def test_quantize_refuses_above_its_range(rt):
    for dtype in (torch.float32, torch.float64):
        w = torch.zeros((1, 4, 1, 40), device="cuda", dtype=dtype)
        w[0, 2, 0, 39] = -7 * 2.0 ** 100
        r = rt.Readout4.quantize(w)
        assert float(r.matvec(torch.ones((1, 4), device="cuda"))[0, 0, 39]) == -7 * 2.0 ** 100
        w[0, 2, 0, 39] = 7.01 * 2.0 ** 100
        with pytest.raises(ValueError, match="2\\*\\*100"):
            rt.Readout4.quantize(w)


def test_from_a_trained_classifier(rt, traces):
    """The read-out of a trained classifier answers as its own weights do, and finds the classifier's best bucket."""
    steps = [1, 2, 3]
    eng = rt.HTMEngine(2, seed_stride=1, seg_capacity=1 << 13)
    cl = rt.classifier.SDRClassifier(2, eng.n_cells, 480, steps=steps, alpha=0.05)
    enc = rt.ScalarEncoder(w=21, minval=0.0, maxval=100.0, n=500, clipInput=True)
    tr = traces["train"]
    for k in range(60):
        v = np.array([tr[k], tr[k + 500]])
        eng.step(torch.tensor(v, device="cuda"))
        prob, _ = cl.compute(eng.get_output("tm_output"), enc.bucket_indices(v), v)
    pat = eng.get_output("tm_output")
    prob = cl.compute(pat, learn=False)[0].cpu().numpy()
    r = cl.readout4()
    assert (r.n_models, r.n_heads, r.n_outputs) == (2, 3, 480)
    assert [int(n) for n in r.live] == [cl.state_summary(s)["max_bucket"] + 1 for s in range(2)]
    got = r.probabilities(pat).cpu().numpy()
    w = cl.export_state("weights").reshape(2, 3, eng.n_cells, 480)
    dense = eng.bitmap_to_dense(pat).astype(bool)
    for s in range(2):
        n = int(r.live[s])
        for y in range(3):
            f = w[s, y][dense[s]]
            # a weight is off by half a step of its group at most, step = max / 7 (bfloat16: 1 + 2^-8)
            top = np.abs(np.pad(f, ((0, 0), (0, 0)))).reshape(len(f), 15, 32).max(-1).repeat(32, -1)
            off = (top / 14 * (1 + 2.0 ** -6)).sum(0)[:n].max()
            p = prob[s, y, :n]
            assert np.all(np.abs(got[s, y, :n] - p) <= p * np.expm1(2 * off + 1e-4))
            assert np.all(got[s, y, n:] == 0)
    one = cl.readout4(1, 1, group=64, steps=[2, 3])
    assert (one.n_models, one.n_heads) == (1, 2)
    both = cl.readout4(group=64)
    nb, ng = 3 * 480 // 2, 8
    a, b = both.records[1], one.records[0]
    assert torch.equal(a[:, 240:nb], b[:, :480])
    assert torch.equal(a[:, nb + 2 * ng:nb + 6 * ng], b[:, 480:480 + 4 * ng])
    for bad in (dict(s0=2), dict(s0=0, n=3), dict(steps=[1, 3]), dict(steps=[9]), dict(steps=[])):
        with pytest.raises(ValueError):
            cl.readout4(**bad)


def test_refusals(rt):
    r, _ = make(rt, 2, 96, 1, 40, 32)
    p = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    for bad in (p.cpu(), p[:1], p[:, :2], p.float(), p.to(torch.int64), p.reshape(-1)):
        with pytest.raises(ValueError):
            r.logits(bad)
    with pytest.raises(ValueError):
        r.logits(p, out=torch.empty((2, 1, 41), device="cuda"))
    for bad in (torch.zeros((2, 96), device="cuda", dtype=torch.float64), torch.zeros((2, 95), device="cuda"),
                torch.zeros((3, 96), device="cuda"), torch.zeros((2, 96))):
        with pytest.raises(ValueError):
            r.matvec(bad)
    with pytest.raises(ValueError, match="gradient"):
        r.matvec(torch.zeros((2, 96), device="cuda", requires_grad=True))
    with torch.no_grad():
        r.matvec(torch.zeros((2, 96), device="cuda", requires_grad=True))
    for bad in (torch.ones(1, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda"), torch.ones(2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            r.probabilities(p, bad)
    odd, _ = make(rt, 1, 33, 1, 40, 32)
    with pytest.raises(ValueError):
        odd.logits(p[:1])
    wide, _ = make(rt, 1, 32, 1, 1025, 32)
    with pytest.raises(rt.HtmError):
        wide.probabilities(p[:1, :1])
    rec = r.records
    for bad in (rec.cpu(), rec[0], rec.to(torch.int32), rec[:, :95].contiguous(), rec[..., :-1]):
        with pytest.raises(ValueError):
            rt.Readout4(bad, 96, 1, 40)
    for bad in (dict(group=16), dict(n_outputs=0), dict(n_heads=65), dict(n_outputs=200)):
        with pytest.raises(ValueError):
            rt.Readout4(rec, **{**dict(n_inputs=96, n_heads=1, n_outputs=40, group=32), **bad})
