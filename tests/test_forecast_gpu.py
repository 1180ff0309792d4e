"""A fleet's streams reordered and forked on the device, and the forecast that
runs read-out, selection and reordering together (harness.model_forecast)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)


@pytest.fixture(scope="module")
def model(rt, traces):
    """A model trained on the first 500 records, and a classifier that learnt its one-step answers beside it."""
    eng = rt.HTMEngine(1, seg_capacity=1 << 15)
    cl = rt.classifier.SDRClassifier(1, eng.n_cells, 480, steps=[1, 2], alpha=0.05)
    enc = rt.ScalarEncoder(w=21, minval=0.0, maxval=100.0, n=500, clipInput=True)
    for v in traces["train"][:500]:
        eng.step(torch.tensor([v], dtype=torch.float64, device="cuda"))
        cl.compute(eng.get_output("tm_output"), enc.bucket_indices(np.array([v])), [v], infer=False)
    eng.status()
    return eng, cl


def values(traces, steps, n, seed):
    rng = np.random.default_rng(seed)
    base = np.asarray(traces["test"][:steps], np.float64)
    v = np.clip(base[:, None] + rng.integers(-4, 5, size=(steps, n)), 0, 100)
    v[rng.random(v.shape) < 0.03] = np.nan
    return v


def same(a, b, streams):
    """Outputs and state of `streams` alike in both engines (the header's last 8 bytes count bytes moved)."""
    for name in ("tm_output", "inf_active", "active_columns", "col_confidence", "buckets"):
        assert torch.equal(a.get_output(name)[streams], b.get_output(name)[streams]), name
    for region in ("tm_bitmaps", "tm_colconf", "tm_patterns", "sp_scalars", "tm_header"):
        x, y = a.export_state(region), b.export_state(region)
        if region == "tm_header":
            x, y = x[:, :-8], y[:, :-8]
        assert np.array_equal(x[streams], y[streams]), region


@pytest.mark.parametrize("beams", [2, 4, 8])
@pytest.mark.parametrize("read", [False, True])
def test_reordered_streams_go_on_as_their_parents(rt, model, traces, beams, read):
    """Every stream's later scores are those of an undisturbed stream that was fed its line of ancestors' values;
    `read`: outputs that change the form of the state are read between."""
    n, before, after = 16, 25, 15
    rng = np.random.default_rng(beams)
    v = values(traces, before + 3 * after, n, 31)
    fl, ref = (rt.HTMEngine.fleet(model[0], n, q_capacity=4096) for _ in range(2))
    fed = np.zeros((0, n))                   # the values each stream's line has lived through
    at = 0
    for part in range(4):
        for _ in range(before if part == 0 else after):
            fl.step(torch.tensor(v[at], device="cuda"))
            fed = np.concatenate((fed, v[at][None]))
            at += 1
            if read and at % 7 == 0:
                fl.get_output("col_confidence")
        if part < 3:
            p = rng.integers(0, beams, (n // beams, beams)).astype(np.int32)
            fl.reorder_streams(torch.from_numpy(p).cuda())
            fed = fed[:, (p + np.arange(n // beams)[:, None] * beams).reshape(-1)]
    for row in fed:
        ref.step(torch.tensor(row, device="cuda"))
    same(fl, ref, slice(None))
    last = torch.tensor(values(traces, 1, n, 5)[0], device="cuda")
    assert torch.equal(fl.step(last), ref.step(last))
    fl.status()


def test_copied_streams_go_on_as_their_sources(rt, model, traces):
    """dst's streams after a fork, with dst and src at different ages, before and after their first step; an index
    outside src leaves a stream alone."""
    n = 6
    v = values(traces, 40, n, 32)
    src, whole = (rt.HTMEngine.fleet(model[0], n, q_capacity=4096) for _ in range(2))
    dst, alone = (rt.HTMEngine.fleet(model[0], 9, q_capacity=4096) for _ in range(2))
    index = np.array([5, 0, 0, -1, 2, 6, 1, 3, 3], np.int32)
    kept = np.array([3, 5])
    taken = np.setdiff1d(np.arange(9), kept)
    w = values(traces, 40, 9, 33)
    t = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    for k in range(20):
        src.step(t(v[k])), whole.step(t(v[k]))
    dst.copy_streams(src, torch.from_numpy(index).cuda())     # dst has not stepped yet
    for k in range(10):
        got = dst.step(t(w[k]))
        alone.step(t(w[k]))
    # dst's streams, run apart from the beginning
    apart = rt.HTMEngine.fleet(model[0], 9, q_capacity=4096)
    for k in range(20):
        apart.step(t(v[k][np.clip(index, 0, n - 1)]))
    for k in range(10):
        want = apart.step(t(w[k]))
    assert torch.equal(got[taken], want[taken])
    same(dst, apart, taken)
    same(dst, alone, kept)
    same(src, whole, slice(None))                             # the sources are as they were
    for k in range(20, 25):
        src.step(t(v[k]))
    src.get_output("col_confidence")
    dst.copy_streams(src, torch.from_numpy(np.clip(index, 0, n - 1)).cuda())
    a, b = dst.export_state("tm_bitmaps"), src.export_state("tm_bitmaps")
    assert np.array_equal(a, b[np.clip(index, 0, n - 1)])
    x = torch.tensor(w[30], device="cuda")
    y = dst.step(x)[1], dst.get_output("tm_output")[1]
    z = src.step(x[1].expand(n).contiguous())
    assert y[0] == z[0] and torch.equal(y[1], src.get_output("tm_output")[0])
    for e in (src, dst):
        e.status()


def test_stream_moves_refused(rt, model):
    fl, other = rt.HTMEngine.fleet(model[0], 6), rt.HTMEngine.fleet(model[0], 4)
    p = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    with pytest.raises(rt.HtmError):
        model[0].reorder_streams(p[:1, :1].contiguous())
    for bad in (p.long(), p.cpu(), p[:2], p.reshape(-1)):
        with pytest.raises(ValueError):
            fl.reorder_streams(bad)
    i = torch.zeros(6, dtype=torch.int32, device="cuda")
    for src, index in ((fl, i), (model[0], i)):
        with pytest.raises(rt.HtmError):
            fl.copy_streams(src, index)
    for bad in (i.long(), i[:5], i.cpu()):
        with pytest.raises(ValueError):
            fl.copy_streams(other, bad)
    yaml = rt.HTMEngine(1, config=rt.default_config(seg_capacity=1 << 14))
    with pytest.raises(rt.HtmError):  # another configuration
        fl.copy_streams(rt.HTMEngine.fleet(yaml, 2), i)
    other.keep_prev_predicted(True)
    with pytest.raises(rt.HtmError):
        fl.copy_streams(other, i)


def test_streams_with_a_distributed_encoder(rt, traces):
    """The RDSE's bucket maps move with their streams."""
    m = rt.HTMEngine(1, config=rt._lib.model_yaml_config(seg_capacity=1 << 15))
    m.run(torch.tensor(traces["train"][:150], dtype=torch.float64, device="cuda").reshape(-1, 1))
    n = 4
    fl, ref = (rt.HTMEngine.fleet(m, n, q_capacity=4096) for _ in range(2))
    rng = np.random.default_rng(3)
    v = rng.uniform(0, 100, (24, n)) + np.arange(n) * 300   # the maps grow apart
    p = np.array([[3, 3, 0, 1]], np.int32)
    for k in range(12):
        fl.step(torch.tensor(v[k], device="cuda"))
        ref.step(torch.tensor(v[k][p[0]], device="cuda"))
    fl.reorder_streams(torch.from_numpy(p).cuda())
    for k in range(12, 24):
        a, b = fl.step(torch.tensor(v[k], device="cuda")), ref.step(torch.tensor(v[k], device="cuda"))
        assert torch.equal(a, b)
    assert np.array_equal(fl.export_state("enc_rdse"), ref.export_state("enc_rdse"))
    same(fl, ref, slice(None))


@pytest.mark.parametrize("source", ["tm_output", "col_confidence"])
def test_forecast_follows_the_best_paths(rt, model, traces, source):
    """The forecast's path and score, against a search that re-runs every kept path from the record with a fleet of
    its own and scores it with the same read-out in plain float64."""
    eng, cl = model
    g, beams, horizon, records = 3, 4, 4, 5
    if source == "tm_output":
        ro = cl.readout4(steps=[1])
    else:
        w = torch.from_numpy(np.random.default_rng(4).standard_normal((1, eng.n_columns, 1, 480)) * 2).cuda()
        ro = rt.Readout4.quantize(w, live=torch.tensor([400], dtype=torch.int32, device="cuda"))
    fl, bf = rt.HTMEngine.fleet(eng, g, q_capacity=4096), rt.HTMEngine.fleet(eng, g * beams, q_capacity=4096)
    v = values(traces, 30, g, 34)
    for row in v[:20]:
        fl.step(torch.tensor(row, device="cuda"))
    out = rt.harness.model_forecast(fl, bf, ro, v[20:20 + records], horizon=horizon, source=source)
    assert out["values"].shape == (records, horizon, g) and out["logp"].shape == out["scores"].shape == (records, g)
    width = (100.0 - 0.0) / 479
    live = int(ro.live[0])

    def answers(e):
        x = e.get_output(source)
        y = (ro.logits(x) if source == "tm_output" else ro.matvec(x))[:, 0, :live].double().cpu().numpy()
        y = y - y.max(1, keepdims=True)
        return y - np.log(np.exp(y).sum(1, keepdims=True))

    # the plain search, all streams' paths in one fleet that starts at the beginning each time
    check = rt.HTMEngine.fleet(eng, g, q_capacity=4096)
    want = [check.step(torch.tensor(row, device="cuda")).cpu().numpy() for row in v[:20 + records]]
    assert np.array_equal(out["scores"], np.stack(want[20:]))
    for t in range(records):
        seen = v[:21 + t]
        paths = [[()] for _ in range(g)]
        total = [[np.float32(0)] for _ in range(g)]
        for h in range(horizon):
            fresh = rt.HTMEngine.fleet(eng, g * beams, q_capacity=4096)
            for row in seen:
                fresh.step(torch.tensor(row.repeat(beams), device="cuda"))
            for k in range(h):
                x = np.array([[paths[s][min(b, len(paths[s]) - 1)][k] * width for b in range(beams)] for s in range(g)])
                fresh.step(torch.tensor(x.reshape(-1), device="cuda"))
            a = answers(fresh).reshape(g, beams, -1)
            for s in range(g):
                n = len(paths[s])
                sc = (a[s, :n] + np.array(total[s], np.float64)[:, None]).astype(np.float32)
                order = np.argsort(-sc.reshape(-1), kind="stable")[:beams]
                paths[s], total[s] = ([paths[s][o // live] + (int(o % live),) for o in order],
                                      [sc.reshape(-1)[o] for o in order])
        for s in range(g):
            best = np.array(paths[s][0]) * width
            assert np.array_equal(out["values"][t, :, s], best), (t, s)
            assert abs(out["logp"][t, s] - total[s][0]) <= horizon * np.spacing(np.float32(abs(total[s][0])))


def test_forecast_refusals_and_no_bucket(rt, model, traces):
    eng, cl = model
    ro = cl.readout4(steps=[1])
    fl, bf = rt.HTMEngine.fleet(eng, 2, q_capacity=4096), rt.HTMEngine.fleet(eng, 6, q_capacity=4096)
    f = rt.harness.model_forecast
    rec = np.array([10.0, 20.0])
    for bad in (dict(fleet=eng), dict(beam_fleet=fl), dict(beam_fleet=rt.HTMEngine.fleet(eng, 5)), dict(readout=cl.readout4()),
                dict(horizon=0), dict(source="sp"), dict(bucket_values=np.zeros(3)), dict(source="col_confidence")):
        with pytest.raises(ValueError):
            f(**{**dict(fleet=fl, beam_fleet=bf, readout=ro, cpu=rec), **bad})
    none = rt.Readout4(ro.records, ro.n_inputs, 1, ro.n_outputs, ro.group, live=torch.zeros(1, dtype=torch.int32, device="cuda"))
    out = f(fl, bf, none, rec, horizon=3)
    assert np.all(np.isnan(out["values"])) and np.all(out["logp"] == -np.inf)
    assert np.all(np.isfinite(f(fl, bf, ro, rec, horizon=1)["values"]))
    assert f(fl, bf, ro, np.zeros((0,)), horizon=2)["values"].shape == (0, 2, 2)
