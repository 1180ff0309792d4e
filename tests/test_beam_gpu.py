"""beam_select / beam_reorder (csrc/beam.hip) against plain numpy in float64.

A score is rounded once, from float64 sums whose own error (some 1e-13 of the
score) may move it across a rounding border: at most one float32 step.  The
places are those of the definition, exactly: the cases' scores are either
equal or much further apart than that."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a GPU", allow_module_level=True)

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def plain(logits, scores, beams, live=None):
    """The definition, one group at a time."""
    x = logits.double().cpu().numpy()
    sc = scores.double().cpu().numpy()
    groups, win, v = x.shape
    o_s = np.full((groups, beams), -np.inf, np.float32)
    o_p = np.minimum(np.arange(beams), win - 1)[None].repeat(groups, 0).astype(np.int32)
    o_b = np.full((groups, beams), -1, np.int32)
    with np.errstate(all="ignore"):
        for g in range(groups):
            n = v if live is None else min(max(int(live[g]), 0), v)
            if n == 0:
                continue
            y = x[g, :, :n]
            m = y.max(1, keepdims=True)
            y = y - m
            s = (y + (sc[g][:, None] - np.log(np.exp(y).sum(1, keepdims=True)))).astype(np.float32)
            s[np.isnan(s)] = -np.inf
            full = np.full((win, v), -np.inf, np.float32)
            full[:, :n] = s
            flat = full.reshape(-1)
            order = np.argsort(-flat, kind="stable")[:beams]
            order = order[flat[order] > -np.inf]
            k = len(order)
            o_s[g, :k], o_p[g, :k], o_b[g, :k] = flat[order], order // v, order % v
    return o_s, o_p, o_b


def check(rt, logits, scores, beams, live=None):
    got = [t.cpu().numpy() for t in rt.beam_select(logits, scores, beams, live=live)]
    want = plain(logits, scores, beams, live)
    assert [a.dtype for a in got] == [np.float32, np.int32, np.int32]
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    fin = np.isfinite(want[0])
    assert np.array_equal(fin, np.isfinite(got[0])) and np.array_equal(got[0][~fin], want[0][~fin])
    assert np.all(np.abs(got[0][fin] - want[0][fin]) <= np.spacing(np.abs(want[0][fin])))
    return got


SIZES = [  # groups, beams_in, beams, outputs
    (1, 1, 1, 1), (1, 1, 8, 480), (3, 8, 8, 480), (5, 4, 3, 7), (2, 1, 64, 5), (2, 64, 64, 3), (1, 64, 64, 1000),
    (7, 5, 5, 479), (33, 8, 8, 481), (2, 3, 17, 1001), (1, 16, 16, 8192), (2, 2, 8, 40000), (1, 1, 5, 100003),
    (3, 32, 32, 2047), (2, 7, 9, 4097), (300, 2, 4, 64), (1, 33, 31, 255), (1, 4, 4, 65536),
    (2, 64, 64, 100), (1, 64, 64, 70000), (2, 3, 7, 1024), (1, 16, 33, 1000), (2, 32, 2, 512), (3, 17, 40, 512),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups,win,beams,v", SIZES)
def test_select(rt, groups, win, beams, v, dtype):
    rng = np.random.default_rng(groups * 1000 + win + beams + v)
    x = torch.from_numpy(rng.standard_normal((groups, win, v)) * 2).to(dtype).cuda()
    s = torch.from_numpy(-rng.random((groups, win)).cumsum(1)).float().cuda()
    check(rt, x, s, beams)
    live = torch.from_numpy(rng.integers(0, v + 1, groups).astype(np.int32)).cuda()
    check(rt, x, s, beams, live)


@pytest.mark.parametrize("v", [40, 480, 3000, 50000])
def test_ties_go_to_the_lowest_place(rt, v):
    rng = np.random.default_rng(v)
    x = torch.from_numpy(rng.integers(0, 3, (4, 6, v))).float().cuda()
    s = torch.zeros((4, 6), device="cuda")
    x[1] = 0.0                      # every continuation alike
    x[2, 1:] = x[2, 0]              # every beam alike
    x[3] = -0.0
    x[3, ::2] = 0.0
    for beams in (1, 6, 64):
        check(rt, x, s, beams)


@pytest.mark.parametrize("v", [9, 480, 20000])
def test_masked_infinite_and_nan(rt, v):
    rng = np.random.default_rng(v)
    x = torch.from_numpy(rng.standard_normal((10, 4, v))).float()
    s = torch.from_numpy(-rng.random((10, 4))).float()
    inf = float("inf")
    x[0] = -inf                                    # nothing left
    x[1, 2] = -inf                                 # one beam without a continuation
    x[2, :, 1:] = -inf                             # one continuation a beam
    x[3, 1, v // 2] = float("nan")                 # the beam's sum is lost, the others' are not
    x[4, 0, 3] = inf
    s[5, 1], s[5, 2] = -inf, float("nan")
    s[6] = -inf
    x[7] = torch.finfo(torch.float32).min          # the type's lowest value everywhere: an even spread
    x[8, :, v // 3:] = torch.finfo(torch.float32).min
    s[9, 3] = inf
    x[9] = x[9] * 1e30
    x, s = x.cuda(), s.cuda()
    for beams in (1, 4, 16):
        got = check(rt, x, s, beams)
        assert np.all(got[2][0] == -1) and np.array_equal(got[1][0], np.minimum(np.arange(beams), 3))
    live = torch.tensor([v, 0, -3, 1, 2, v + 5, v, v // 2, v // 3, 1], dtype=torch.int32, device="cuda")
    check(rt, x, s, 8, live)


@pytest.mark.parametrize("win,v", [(1, 200), (64, 256), (8, 480), (16, 1000), (3, 2500), (5, 60000)])
def test_more_candidates_than_a_short_list(rt, win, v):
    """Every 64th output low, in order or against it: nearly all candidates lie above what 64 of them are sure to reach."""
    rng = np.random.default_rng(v)
    x = rng.standard_normal((4, win, v))
    x[1] = np.sort(x[1], -1)
    x[2] = np.sort(x[2], -1)[:, ::-1]
    x[3] = np.round(x[3])
    x[..., 5::64] -= 60
    x = torch.from_numpy(x.copy()).float().cuda()
    s = torch.from_numpy(-rng.random((4, win))).float().cuda()
    for beams in (64, 33, 2):
        check(rt, x, s, beams)


def test_calls_at_once(rt):
    """Selections and in-place moves on two streams at the same time."""
    rng = np.random.default_rng(5)
    work = []
    for k in range(2):
        x = torch.from_numpy(rng.standard_normal((64, 4, 30000))).float().cuda()
        s = torch.from_numpy(-rng.random((64, 4))).float().cuda()
        state = torch.from_numpy(rng.integers(0, 1 << 30, (256, 5000))).cuda()
        want = rt.beam_select(x, s, 4)
        work.append((x, s, state, want, rt.beam_reorder([state], want[1], out=[torch.empty_like(state)])[0]))
    torch.cuda.synchronize()
    got = []
    for x, s, state, _, _ in work:
        with torch.cuda.stream(torch.cuda.Stream()):
            r = rt.beam_select(x, s, 4)
            got.append((r, rt.beam_reorder([state.clone()], r[1])[0]))
    torch.cuda.synchronize()
    for (r, moved), (_, _, _, want, at) in zip(got, work):
        assert all(torch.equal(p, q) for p, q in zip(r, want)) and torch.equal(moved, at)


def test_reorder_in_place_captured_into_a_graph(rt):
    rng = np.random.default_rng(6)
    first = torch.from_numpy(rng.integers(0, 99, (24, 1037), dtype=np.uint8)).cuda()
    a, b = first.clone(), first.clone()
    p = torch.from_numpy(rng.integers(0, 8, (3, 8)).astype(np.int32)).cuda()
    with torch.cuda.stream(torch.cuda.Stream()):
        rt.beam_reorder([b.clone()], p)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rt.beam_reorder([a], p)
    for _ in range(5):
        p.copy_(torch.from_numpy(rng.integers(0, 8, (3, 8)).astype(np.int32)))
        g.replay()
        rt.beam_reorder([b], p)
        torch.cuda.synchronize()
        assert torch.equal(a, b)


def test_scores_of_very_different_size(rt):
    x = torch.zeros((1, 3, 8), device="cuda")
    x[0, 0, 5], x[0, 1, 2] = 80.0, -300.0
    s = torch.tensor([[-1e6, -1e-3, -3.4e38]], device="cuda")
    check(rt, x, s, 24)


def test_strides_streams_and_many_groups(rt):
    rng = np.random.default_rng(1)
    big = torch.from_numpy(rng.standard_normal((6, 4, 7, 480))).float().cuda()  # [groups, beams, heads, outputs]
    s = torch.from_numpy(-rng.random((6, 4))).float().cuda()
    for view in (big[:, :, 3], big[:, :, 6, 1:], big[:, :, 2, ::2], big[::2, :, 0], big[:, :1, 0].expand(6, 4, 480)):
        sc = s[:view.shape[0]]
        check(rt, view, sc, 5)
        check(rt, view, sc.t().contiguous().t(), 5)
    assert rt.beam_select(big[:0, :, 0], s[:0], 4)[0].shape == (0, 4)
    a = rt.beam_select(big[:, :, 0], s, 4)
    torch.cuda.synchronize()
    for _ in range(2):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            b = rt.beam_select(big[:, :, 0], s, 4)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    x = torch.from_numpy(rng.standard_normal((70000, 1, 3))).float().cuda()  # more groups than one grid dimension holds
    check(rt, x, torch.zeros((70000, 1), device="cuda"), 2)
    n = (1 << 20) + 5                                                        # and than one launch takes
    x = torch.from_numpy(rng.standard_normal((n, 1, 2))).float().cuda()
    got = rt.beam_select(x, torch.zeros((n, 1), device="cuda"), 1)
    assert torch.equal(got[2][:, 0].long(), x[:, 0].argmax(1)) and torch.all(got[1] == 0)


@pytest.mark.parametrize("v", [480, 30000])
def test_select_captured_into_graphs(rt, v):
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((3, 4, v))).float().cuda()
    s = torch.zeros((3, 4), device="cuda")
    state = [torch.from_numpy(rng.integers(0, 99, (12, 37))).cuda(), torch.zeros((3, 4, 5), device="cuda")]
    out = [torch.empty_like(t) for t in state]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        rt.beam_reorder(state, rt.beam_select(x, s, 4)[1], out=out)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = rt.beam_select(x, s, 4)
            rt.beam_reorder(state, r[1], out=out)
        graphs.append((g, r))
    for k in range(6):
        x.copy_(torch.from_numpy(rng.standard_normal((3, 4, v))))
        g, r = graphs[k % 2]
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = rt.beam_select(x, s, 4)
        assert all(torch.equal(p, q) for p, q in zip(r, want))
        assert all(torch.equal(p, q) for p, q in zip(got, rt.beam_reorder([t.clone() for t in state], want[1])))


def test_select_refusals(rt):
    x = torch.zeros((2, 3, 5), device="cuda")
    s = torch.zeros((2, 3), device="cuda")
    for args in ((x.cpu(), s, 2), (x.double(), s, 2), (x[0], s, 2), (x, s.cpu(), 2), (x, s[:1], 2), (x, s.double(), 2),
                 (x, s, 0), (x, s, 65), (x[..., :0], s, 2), (x[:, :0], s[:, :0], 2),
                 (torch.zeros((1, 65, 2), device="cuda"), torch.zeros((1, 65), device="cuda"), 2)):
        with pytest.raises(ValueError):
            rt.beam_select(*args)
    with pytest.raises(ValueError, match="gradient"):
        rt.beam_select(x.clone().requires_grad_(), s, 2)
    for live in (torch.ones(2, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            rt.beam_select(x, s, 2, live=live)


# ------------------------------------------------------------------- reorder
def parents(rng, groups, beams, kind):
    if kind == "any":
        return rng.integers(0, beams, (groups, beams))
    if kind == "turned":
        return np.roll(np.arange(beams), 1)[None].repeat(groups, 0)
    if kind == "one":
        return np.full((groups, beams), beams - 1)
    if kind == "same":
        return np.arange(beams)[None].repeat(groups, 0)
    p = rng.integers(-2, beams + 2, (groups, beams))  # "outside": counts as the row itself
    p[0, 0], p[-1, -1] = 2 ** 31 - 1, -2 ** 31
    return p


@pytest.mark.parametrize("kind", ["any", "turned", "one", "same", "outside"])
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 8), (5, 3), (64, 8), (2, 64), (3, 33), (9, 16), (2, 17)])
def test_reorder(rt, groups, beams, kind):
    rng = np.random.default_rng(groups + beams)
    p = parents(rng, groups, beams, kind)
    rows = groups * beams
    eff = np.where((p >= 0) & (p < beams), p, np.arange(beams))
    at = (eff + np.arange(groups)[:, None] * beams).reshape(-1)
    raw = [rng.integers(0, 256, (rows, n), dtype=np.uint8) for n in (1, 3, 4, 8, 16, 37, 296, 1024, 12288 + 4)]
    bufs = [torch.from_numpy(b).cuda() for b in raw]
    bufs.append(torch.from_numpy(raw[3].copy().view(np.float64).reshape(groups, beams)).cuda())  # a number a row
    raw = raw + [raw[3].copy()]
    # rows that begin at odd addresses, with bytes around them that stay
    flat = torch.full((rows * 20 + 40,), 77, dtype=torch.uint8, device="cuda")
    odd = flat[13:13 + rows * 20].view(rows, 20)
    odd.copy_(bufs[5][:, :20])
    bufs.append(odd)
    raw.append(raw[5][:, :20].copy())
    parent = torch.from_numpy(p.astype(np.int32)).cuda()
    outs = [torch.empty_like(b) for b in bufs]
    keep = [b.clone() for b in bufs]
    got = rt.beam_reorder(bufs, parent, out=outs)
    for a, b, c, k in zip(got, raw, bufs, keep):
        assert torch.equal(c.view(torch.uint8), k.view(torch.uint8))  # (some bytes make NaNs)
        assert np.array_equal(a.contiguous().cpu().numpy().view(np.uint8).reshape(rows, -1), b[at])
    assert rt.beam_reorder(bufs, parent) == bufs
    for a, b in zip(bufs, raw):
        assert np.array_equal(a.contiguous().cpu().numpy().view(np.uint8).reshape(rows, -1), b[at])
    assert torch.all(flat[:13] == 77) and torch.all(flat[13 + rows * 20:] == 77)


def test_reorder_mixed_and_empty(rt):
    a, b = torch.arange(6, device="cuda"), torch.arange(6, device="cuda") * 10
    o = torch.empty_like(b)
    p = torch.tensor([[1, 1], [1, 0], [0, 0]], dtype=torch.int32, device="cuda")
    assert [t.tolist() for t in rt.beam_reorder([a, b], p, out=[a, o])] == [[1, 1, 3, 2, 4, 4], [10, 10, 30, 20, 40, 40]]
    empty = torch.zeros((6, 0), device="cuda")
    rt.beam_reorder([a, empty], p)
    rt.beam_reorder([torch.zeros((0, 4), device="cuda")], p[:0])


def test_reorder_refusals(rt):
    p = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    a = torch.zeros((12, 8), device="cuda")
    for bad in (([a], p.long()), ([a], p.cpu()), ([a], p.reshape(-1)), ([], p), ([a[:11]], p), ([a.t()], p), ([a.cpu()], p),
                ([torch.zeros((3, 4), device="cuda")] * 33, p), ([a], p, [a.double()]), ([a], p, [a, a]),
                ([a], torch.zeros((1, 65), dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            rt.beam_reorder(*bad)
    big = torch.zeros(12 * 8 + 8, device="cuda")
    for bad in (([a, a], p), ([big[:96].view(12, 8)], p, [big[8:].view(12, 8)]),
                ([a, big[:96].view(12, 8)], p, [big[:96].view(12, 8), torch.zeros((12, 8), device="cuda")]),
                ([p.view(12)], p)):
        with pytest.raises(rt.HtmError):
            rt.beam_reorder(*bad)
