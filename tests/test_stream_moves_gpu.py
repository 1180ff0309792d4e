"""What a move of a fleet's streams must not lose or accept (HTMEngine.reorder_streams, copy_streams,
harness.model_forecast)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

OVERFLOW = 16  # htm_tm_header.error: qualifying-segment list overflow


def trained(rt, traces, steps=120, first=0):
    eng = rt.HTMEngine(1, seg_capacity=1 << 14)
    for v in traces["train"][first:first + steps]:
        eng.step(torch.tensor([v], dtype=torch.float64, device="cuda"))
    return eng


@pytest.fixture(scope="module")
def model(rt, traces):
    return trained(rt, traces)


def flag(rt, fleet, stream, bits):
    """The stream's header as an overflow leaves it."""
    h = fleet.tm_header(stream)
    h.error |= bits
    fleet.import_state("tm_header", np.frombuffer(bytes(h), np.uint8)[None], stream)


def flags(fleet):
    return [fleet.tm_header(s).error for s in range(fleet.n_streams)]


def step(fleet, value):
    fleet.step(torch.full((fleet.n_streams,), float(value), dtype=torch.float64, device="cuda"))


@pytest.mark.parametrize("beams", [1, 3, 6])
def test_flags_stay_with_a_stream_that_is_reordered(rt, model, beams):
    fl = rt.HTMEngine.fleet(model, 6, q_capacity=4096)
    step(fl, 30)
    flag(rt, fl, 1, OVERFLOW)
    flag(rt, fl, 5, 2)
    parent = np.zeros((6 // beams, beams), np.int32)   # the first stream of a group is the parent of all
    parent[-1, -1] = 99                                # outside: the stream itself
    fl.reorder_streams(torch.from_numpy(parent).cuda())
    at = (parent % 99 + np.arange(6 // beams)[:, None] * beams).reshape(-1)
    old = [0, OVERFLOW, 0, 0, 0, 2]
    assert flags(fl) == [old[s] | (old[at[s]] if s < 5 else 0) for s in range(6)]
    with pytest.raises(rt.HtmError, match="q_capacity|queue full"):
        fl.status()
    if beams > 1:  # a flagged parent's children are flagged too
        fl.reorder_streams(torch.full((6 // beams, beams), 1, dtype=torch.int32, device="cuda"))
        assert flags(fl)[0] == OVERFLOW
    step(fl, 31)
    with pytest.raises(rt.HtmError):
        fl.status()


def test_flags_stay_with_a_stream_that_is_copied_to(rt, model):
    src, dst = rt.HTMEngine.fleet(model, 2, q_capacity=4096), rt.HTMEngine.fleet(model, 5, q_capacity=4096)
    step(src, 30), step(dst, 40)
    flag(rt, dst, 3, OVERFLOW)
    index = torch.tensor([0, 1, -1, 0, 7], dtype=torch.int32, device="cuda")
    dst.copy_streams(src, index)
    assert flags(dst) == [0, 0, 0, OVERFLOW, 0] and flags(src) == [0, 0]
    flag(rt, src, 1, 1)
    dst.copy_streams(src, index)
    assert flags(dst) == [0, 1, 0, OVERFLOW, 0]
    with pytest.raises(rt.HtmError):
        dst.status()


@pytest.mark.parametrize("horizon", [2, 4])
def test_a_forecast_raises_for_a_beam_that_was_replaced(rt, model, horizon):
    """An overflow of an early look-ahead step: the beam's state is replaced by forks and reorders many times after."""
    w = torch.from_numpy(np.random.default_rng(3).standard_normal((1, model.n_columns, 1, 480))).cuda()
    ro = rt.Readout4.quantize(w)
    fl, bf = rt.HTMEngine.fleet(model, 2, q_capacity=4096), rt.HTMEngine.fleet(model, 8, q_capacity=4096)
    records = np.array([20.0, 30.0, 25.0])
    rt.harness.model_forecast(fl, bf, ro, records, horizon=horizon, source="col_confidence")
    for stream in (0, 3, 6):
        flag(rt, bf, stream, OVERFLOW)
        with pytest.raises(rt.HtmError, match="q_capacity"):
            rt.harness.model_forecast(fl, bf, ro, records, horizon=horizon, source="col_confidence")
        for s in range(8):                             # (its children are flagged too)
            h = bf.tm_header(s)
            h.error = 0
            bf.import_state("tm_header", np.frombuffer(bytes(h), np.uint8)[None], s)
    rt.harness.model_forecast(fl, bf, ro, records, horizon=horizon, source="col_confidence")


def test_fleets_of_different_models_are_refused(rt, model, traces, tmp_path):
    """Alike in configuration: trained on other records, and one model before and after more training."""
    index = torch.zeros(3, dtype=torch.int32, device="cuda")
    other = trained(rt, traces, first=400)
    grown = trained(rt, traces)
    early = rt.HTMEngine.fleet(grown, 3, q_capacity=4096)
    for v in traces["train"][120:150]:
        grown.step(torch.tensor([v], dtype=torch.float64, device="cuda"))
    late = rt.HTMEngine.fleet(grown, 3, q_capacity=4096)
    fl = rt.HTMEngine.fleet(model, 3, q_capacity=4096)
    for dst, src in ((fl, rt.HTMEngine.fleet(other, 2, q_capacity=4096)), (early, late), (late, early)):
        assert dst.model_id() != src.model_id()
        with pytest.raises(rt.HtmError, match="models differ"):
            dst.copy_streams(src, index)
    w = torch.from_numpy(np.random.default_rng(3).standard_normal((1, model.n_columns, 1, 480))).cuda()
    ro = rt.Readout4.quantize(w)
    step(fl, 10)
    before = fl.export_state("tm_header")
    with pytest.raises(ValueError, match="one model"):
        rt.harness.model_forecast(fl, rt.HTMEngine.fleet(other, 6, q_capacity=4096), ro, np.array([20.0]), horizon=2,
                                  source="col_confidence")
    assert np.array_equal(before, fl.export_state("tm_header"))   # refused before the first step
    with pytest.raises(rt.HtmError):
        model.model_id()


def test_fleets_of_one_model_are_not(rt, model, traces, tmp_path):
    """Built at different times, with different list capacities, stepped, saved and loaded, from models equal in
    content: one identity."""
    index = torch.zeros(3, dtype=torch.int32, device="cuda")
    a = rt.HTMEngine.fleet(model, 3, q_capacity=4096)
    for v in (10, 50, 90, 20, 30, 40, 50, 60, 70):
        step(a, v)                                       # (a flush of the deferred writes among them)
    a.save(str(tmp_path / "fleet"))
    loaded = rt.HTMEngine.load(str(tmp_path / "fleet"))
    again = trained(rt, traces)                          # the same training once more
    b, c = rt.HTMEngine.fleet(model, 2, q_capacity=2048), rt.HTMEngine.fleet(again, 5, q_capacity=4096)
    ids = {e.model_id() for e in (a, b, c, loaded)}
    assert len(ids) == 1
    for src in (b, c, loaded):
        a.copy_streams(src, index)
    # another model's state imported makes another fleet of it, its own makes it this one again
    own = b.export_state("tm_seg_perm", 0, 1)
    b.import_state("tm_seg_perm", np.zeros_like(own))
    assert b.model_id() not in ids
    with pytest.raises(rt.HtmError, match="models differ"):
        a.copy_streams(b, index)
    b.import_state("tm_seg_perm", own)
    assert b.model_id() in ids
    a.copy_streams(b, index)
    a.status()


def test_moves_are_not_captured(rt, model):
    """The state's form when a move is called decides what moves; a replay would not know it."""
    fl, src = rt.HTMEngine.fleet(model, 4, q_capacity=4096), rt.HTMEngine.fleet(model, 2, q_capacity=4096)
    step(fl, 30), step(src, 40)
    p = torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    before = fl.export_state("tm_bitmaps")
    x = torch.ones(8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.mul_(2.0)
        for move in (lambda: fl.reorder_streams(p), lambda: fl.copy_streams(src, i)):
            with pytest.raises(rt.HtmError, match="captured"):
                move()
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.all(x == 2.0 ** (k + 1))
    assert np.array_equal(fl.export_state("tm_bitmaps"), before)
    fl.reorder_streams(p)
    assert np.array_equal(fl.export_state("tm_bitmaps"), before[[1, 0, 3, 3]])
