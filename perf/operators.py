"""What the read-out and beam operators are measured on.

Kinds of case:

* "logits" / "probabilities" -- Readout4 on word bitmaps of TM cells (the
  SDRClassifier's product with 4-bit weights and one scale per group of
  buckets): `rows` patterns, `models` matrices of `inputs` cells x `heads`
  look-ahead steps x `outputs` buckets;
* "matvec" -- Readout4 on vectors of numbers (column confidences, or cells'
  activity), types float32 / float16 / bfloat16, `filled` of them not zero;
* "select" -- beam_select: the best `beams` of `beams_in` x `outputs`
  continuations of each of `groups` streams;
* "reorder" -- beam_reorder: the beams' states (cell bitmaps, column
  confidences, pattern history, header) gathered by parent;
* "step" -- the two together, as one look-ahead step of a forecast runs them.
"""
import math

import torch

own = False

#: rows of a pattern history and columns of one row, and bytes of a header, of a TM state
HISTORY, ACTIVE, HEADER = 32, 64, 296


def _readout(name, kind, rows, models, inputs, heads, outputs, group=32, **more):
    return dict(name=name, kind=kind, rows=rows, models=models, inputs=inputs, heads=heads, outputs=outputs,
                group=group, **more)


def _select(name, groups, beams_in, beams, outputs, dtype="float32"):
    return dict(name=name, kind="select", groups=groups, beams_in=beams_in, beams=beams, outputs=outputs, dtype=dtype)


def listed():
    return [
        # one stream's classifier answer: 2048 columns x 12 cells, steps 1..7, 480 buckets
        _readout("logits: one stream", "logits", 1, 1, 24576, 7, 480),
        # a fleet's one-step answer from the model that it shares
        _readout("logits: fleet, shared", "logits", 4096, 1, 24576, 1, 480),
        # streams that were trained apart, each with matrices of its own
        _readout("logits: own matrices", "logits", 256, 256, 24576, 7, 480),
        # 32 cells a column and the 1000 buckets of the distributed encoder; eight beams a matrix
        _readout("probabilities: 32 cells", "probabilities", 64, 8, 65536, 1, 1000, group=64),
        # one stream's column confidences (topDownOut) to the next value's bucket: few columns have any
        _readout("matvec: confidences", "matvec", 1, 1, 2048, 1, 480, dtype="float32", filled=0.06),
        # a few streams' cell activities, averaged over time, through all seven steps' matrices: none is zero
        _readout("matvec: eight rows", "matvec", 8, 1, 24576, 7, 480, dtype="bfloat16", filled=1.0),
        # one stream's eight beams
        _select("select: one stream", 1, 8, 8, 480),
        # a fleet's beams
        _select("select: fleet", 4096, 8, 8, 480),
        # a joint vocabulary of several fields' buckets, wider beams
        _select("select: wide vocabulary", 4, 16, 16, 32768, dtype="bfloat16"),
        # one stream's beams change places
        dict(name="reorder: one stream", kind="reorder", groups=1, beams=8, cells=24576, columns=2048),
        # a fleet's
        dict(name="reorder: fleet", kind="reorder", groups=1024, beams=8, cells=24576, columns=2048),
        # one look-ahead step of a fleet's forecast
        dict(name="step: fleet", kind="step", groups=512, beams=8, cells=24576, columns=2048, outputs=480),
    ]


def _spread(rng, low, high):
    """A whole number of low..high, spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["logits", "logits", "probabilities", "matvec", "select", "select", "reorder", "step"])
    if kind in ("logits", "probabilities", "matvec"):
        heads = rng.choice([1, 1, 3, 7])
        outputs = rng.choice([_spread(rng, 2, 1000), 480, rng.randint(401, 503)])
        group = rng.choice([32, 64, 128])
        if kind == "matvec":
            return dict(kind=kind, rows=_spread(rng, 1, 12), models=1, inputs=_spread(rng, 33, 24576), heads=heads,
                        outputs=outputs, group=group, dtype=rng.choice(["float32", "float16", "bfloat16"]),
                        filled=rng.choice([0.06, round(rng.uniform(0.02, 1.0), 3), 1.0]))
        # 64 columns (the smallest pooler) up to 2048, 2 to 32 cells each
        inputs = 64 * _spread(rng, 1, 32) * rng.choice([2, 4, 12, 32])
        models = rng.choice([1, 1, _spread(rng, 2, 32)])
        rows = models * _spread(rng, 1, max(1, (1024 if heads == 1 else 256) // models))
        return dict(kind=kind, rows=rows, models=models, inputs=inputs, heads=heads, outputs=outputs, group=group)
    if kind == "select":
        outputs = rng.choice([_spread(rng, 2, 1000), _spread(rng, 1001, 40000)])
        beams = _spread(rng, 1, 32)
        groups = _spread(rng, 1, max(1, min(4096, 8000000 // (beams * outputs))))
        return dict(kind=kind, groups=groups, beams_in=rng.choice([beams, beams, 1]), beams=beams, outputs=outputs,
                    dtype=rng.choice(["float32", "float32", "float16", "bfloat16"]))
    columns = 64 * _spread(rng, 1, 32)
    cells = columns * rng.choice([2, 4, 12, 32])
    beams = _spread(rng, 2, 32)
    if kind == "reorder":
        return dict(kind=kind, groups=_spread(rng, 1, max(1, 4096 // beams)), beams=beams, cells=cells, columns=columns)
    return dict(kind=kind, groups=_spread(rng, 1, max(1, 2048 // beams)), beams=beams, cells=cells, columns=columns,
                outputs=rng.choice([480, rng.randint(40, 1000)]))


# ---------------------------------------------------------------- inputs
def _up(n, to):
    return -(-n // to) * to


def _layout(c):
    """(padded outputs a head, scale groups a head, bytes of codes, bytes of a record): a record holds one input's
    weights, all heads' 4-bit codes (8 stands for zero, the lower half of a byte first), then all heads' bfloat16 scales."""
    heads = c["heads"]
    padded = _up(c["outputs"], 32)
    groups = -(-padded // c["group"])
    return padded, groups, heads * padded // 2, _up(heads * padded // 2 + 2 * heads * groups, 64)


def _records(c, gen):
    """Matrices as training leaves them: weights around zero, a few buckets of each input's groups larger."""
    padded, groups, codes, pitch = _layout(c)
    models, inputs, heads = c["models"], c["inputs"], c["heads"]
    rec = torch.randint(-2 ** 31, 2 ** 31, (models, inputs, pitch // 4), dtype=torch.int32, device="cuda", generator=gen)
    rec = rec.view(torch.uint8)
    for m in range(0, models, 16):  # a part at a time: the largest case's scales would take as much again
        s = torch.rand((min(16, models - m), inputs, heads * groups), device="cuda", generator=gen)
        s = (0.002 + 0.05 * s ** 4).to(torch.bfloat16)
        rec[m:m + 16, :, codes:codes + 2 * heads * groups] = s.contiguous().view(torch.uint8)
    return rec


def _pattern(rows, inputs, columns, gen):
    """TM outputs as word bitmaps: 40 active columns; in two steps of five they burst, else one cell of each is active
    and 20 to 200 cells are predicted."""
    per = inputs // columns
    active = min(40, columns)
    dense = torch.zeros((rows, columns, per), dtype=torch.bool, device="cuda")
    for at in range(0, rows, 512):
        n = min(512, rows - at)
        part = dense[at:at + n]
        cols = torch.rand((n, columns), device="cuda", generator=gen).argsort(1)[:, :active]
        one = torch.randint(0, per, (n, active), device="cuda", generator=gen)
        bursts = torch.rand((n, 1, 1), device="cuda", generator=gen) < 0.4
        cells = (torch.arange(per, device="cuda") == one[..., None]) | bursts
        part.scatter_(1, cols[..., None].expand(-1, -1, per), cells)
        share = (20 + 180 * torch.rand((n, 1, 1), device="cuda", generator=gen)) / inputs
        part |= (torch.rand((n, columns, per), device="cuda", generator=gen) < share) & ~bursts
    bits = dense.reshape(rows, inputs // 32, 32).to(torch.int64) << torch.arange(32, device="cuda")
    words = bits.sum(2)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _columns(c):
    """Columns of `inputs` cells: 32, 12, 4 or 2 cells each (64 columns at least)."""
    return next(c["inputs"] // k for k in (32, 12, 4, 2) if c["inputs"] % (64 * k) == 0)


def _logits(groups, beams, outputs, dtype, gen):
    """A classifier's answers: a hill around one bucket, a low plain elsewhere."""
    at = torch.rand((groups, beams, 1), device="cuda", generator=gen) * outputs
    wide = 2 + 10 * torch.rand((groups, beams, 1), device="cuda", generator=gen)
    x = torch.randn((groups, beams, outputs), device="cuda", generator=gen) * 0.5
    x += 6 * torch.exp(-((torch.arange(outputs, device="cuda") - at) / wide) ** 2)
    return x.to(dtype)


def _scores(groups, beams, gen):
    return -torch.cumsum(torch.rand((groups, beams), device="cuda", generator=gen), 1)


def _states(rows, cells, columns, gen):
    """What a stream carries from step to step: four cell bitmaps, column confidences, pattern history, header."""
    ints = dict(device="cuda", generator=gen)
    return [torch.randint(-2 ** 31, 2 ** 31, (rows, 4, cells // 32), dtype=torch.int32, **ints),
            torch.rand((rows, columns), **ints),
            torch.randint(-2 ** 15, 2 ** 15, (rows, HISTORY, ACTIVE), dtype=torch.int16, **ints),
            torch.randint(0, 256, (rows, HEADER), dtype=torch.uint8, **ints)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, kind, s = case, case["kind"], {"case": dict(case)}
    if own:
        import _pkg
        s["rt"] = _pkg.load()
    if kind in ("logits", "probabilities", "matvec"):
        s["records"] = _records(c, gen)
        if own:  # the handle that a program keeps with its matrices
            s["readout"] = s["rt"].Readout4(s["records"], c["inputs"], c["heads"], c["outputs"], c["group"])
    if kind in ("logits", "probabilities"):
        s["pattern"] = _pattern(c["rows"], c["inputs"], _columns(c), gen)
    if kind == "probabilities":  # buckets seen so far, of each matrix
        s["live"] = torch.randint(max(1, c["outputs"] // 2), c["outputs"] + 1, (c["models"],), dtype=torch.int32,
                                  device="cuda", generator=gen)
    if kind == "matvec":
        x = torch.rand((2, c["rows"], c["inputs"]), device="cuda", generator=gen)
        s["x"] = torch.where(x[0] < c["filled"], x[1], torch.zeros_like(x[1])).to(getattr(torch, c["dtype"]))
    if kind == "select":
        s["logits"] = _logits(c["groups"], c["beams_in"], c["outputs"], getattr(torch, c["dtype"]), gen)
        s["scores"] = _scores(c["groups"], c["beams_in"], gen)
        s["live"] = torch.randint(max(1, c["outputs"] // 2), c["outputs"] + 1, (c["groups"],), dtype=torch.int32,
                                  device="cuda", generator=gen)
    if kind == "reorder":
        s["states"] = _states(c["groups"] * c["beams"], c["cells"], c["columns"], gen)
        s["out"] = [torch.empty_like(t) for t in s["states"]]
        # the better beams have more children
        u = torch.rand((c["groups"], c["beams"]), device="cuda", generator=gen)
        s["parent"] = (c["beams"] * u * u).to(torch.int32).clamp_(max=c["beams"] - 1)
    if kind == "step":
        s["logits"] = _logits(c["groups"], c["beams"], c["outputs"], torch.float32, gen)
        s["scores"] = _scores(c["groups"], c["beams"], gen)
        s["states"] = _states(c["groups"] * c["beams"], c["cells"], c["columns"], gen)
        s["out"] = [torch.empty_like(t) for t in s["states"]]
    return s


# ---------------------------------------------------------------- the plain forms
def _weights(c, rec):
    """float32 weights [..., heads, outputs] of records [..., pitch]."""
    padded, groups, codes, _ = _layout(c)
    heads = c["heads"]
    b = rec[..., :codes]
    q = torch.stack((b & 15, b >> 4), -1).reshape(*rec.shape[:-1], heads, padded).float() - 8
    s = rec[..., codes:codes + 2 * heads * groups].contiguous().view(torch.bfloat16).float()
    s = s.reshape(*rec.shape[:-1], heads, groups).repeat_interleave(c["group"], -1)[..., :padded]
    return (q * s)[..., :c["outputs"]]


def _plain_logits(c, rec, pattern):
    bits = (pattern[..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    bits = bits.reshape(pattern.shape[0], -1)
    if rec.shape[0] == 1 and pattern.shape[0] >= 64:  # many rows of one matrix: a product costs less than their rows apart
        return _plain_matvec(c, rec, bits)
    row, cell = bits.nonzero(as_tuple=True)
    w = _weights(c, rec[row // (pattern.shape[0] // rec.shape[0]), cell])
    y = torch.zeros((pattern.shape[0], c["heads"], c["outputs"]), device="cuda")
    return y.index_add_(0, row, w)


def _plain_probabilities(c, rec, pattern, live):
    y = _plain_logits(c, rec, pattern)
    live = live.repeat_interleave(pattern.shape[0] // rec.shape[0])
    y = y.masked_fill(torch.arange(c["outputs"], device="cuda") >= live[:, None, None], -math.inf)
    e = torch.exp(y - y.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_matvec(c, rec, x):
    w = _weights(c, rec[0]).reshape(c["inputs"], -1)
    return (x.float() @ w).reshape(x.shape[0], c["heads"], c["outputs"])


def _plain_select(logits, scores, beams, live):
    """Scores in 64 bits up to their one rounding: two next to each other change places otherwise."""
    groups, into, outputs = logits.shape
    x = logits.double()
    if live is not None:
        x = x.masked_fill(torch.arange(outputs, device="cuda") >= live[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x - top
    total = torch.log(torch.exp(x).sum(-1, keepdim=True))
    cand = (x + (scores.double()[..., None] - total)).float().reshape(groups, into * outputs)
    cand = torch.where(cand.isnan(), torch.full_like(cand, -math.inf), cand) + 0.0
    bits = cand.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * 2 ** 32 + (2 ** 31 - torch.arange(into * outputs, device="cuda"))
    if key.shape[1] < beams:
        key = torch.nn.functional.pad(key, (0, beams - key.shape[1]), value=-2 ** 62)
        cand = torch.nn.functional.pad(cand, (0, beams - cand.shape[1]), value=-math.inf)
    at = key.topk(beams, dim=1).indices
    best = cand.gather(1, at)
    none = best == -math.inf
    slot = torch.arange(beams, device="cuda").clamp(max=into - 1)
    return best, torch.where(none, slot, at // outputs).int(), torch.where(none, -1, at % outputs).int()


def _plain_reorder(states, parent, out):
    at = (parent + torch.arange(parent.shape[0], device="cuda")[:, None] * parent.shape[1]).reshape(-1)
    for t, o in zip(states, out):
        o.copy_(t[at])
    return out


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        rt = s["rt"]
        if kind == "logits":
            return s["readout"].logits(s["pattern"])
        if kind == "probabilities":
            return s["readout"].probabilities(s["pattern"], s["live"])
        if kind == "matvec":
            return s["readout"].matvec(s["x"])
        if kind == "select":
            return rt.beam_select(s["logits"], s["scores"], c["beams"], live=s["live"])
        if kind == "reorder":
            return rt.beam_reorder(s["states"], s["parent"], out=s["out"])
        scores, parent, bucket = rt.beam_select(s["logits"], s["scores"], c["beams"])
        return scores, parent, bucket, rt.beam_reorder(s["states"], parent, out=s["out"])
    if kind == "logits":
        return _plain_logits(c, s["records"], s["pattern"])
    if kind == "probabilities":
        return _plain_probabilities(c, s["records"], s["pattern"], s["live"])
    if kind == "matvec":
        return _plain_matvec(c, s["records"], s["x"])
    if kind == "select":
        return _plain_select(s["logits"], s["scores"], c["beams"], s["live"])
    if kind == "reorder":
        return _plain_reorder(s["states"], s["parent"], s["out"])
    scores, parent, bucket = _plain_select(s["logits"], s["scores"], c["beams"], None)
    return scores, parent, bucket, _plain_reorder(s["states"], parent, s["out"])


# ---------------------------------------------------------------- in 64 bits
def _exact_logits(c, rec, dense):
    """float64 sums, a slice of the inputs at a time; dense: [rows, inputs] multipliers."""
    padded, groups, codes, _ = _layout(c)
    heads, models, rows = c["heads"], rec.shape[0], dense.shape[0]
    y = torch.zeros((models, rows // models, heads * padded), dtype=torch.float64, device="cuda")
    for m in range(models):
        x = dense[m * (rows // models):(m + 1) * (rows // models)]
        used = x.ne(0).any(0).nonzero()[:, 0]
        for part in used.split(2048):
            r = rec[m, part]
            q = torch.empty((len(part), heads * padded), dtype=torch.float64, device="cuda")
            q[:, 0::2] = (r[:, :codes] % 16).double()
            q[:, 1::2] = torch.div(r[:, :codes], 16, rounding_mode="floor").double()
            s = r[:, codes:codes + 2 * heads * groups].contiguous().view(torch.bfloat16).double()
            of = torch.arange(heads * padded, device="cuda")
            of = of // padded * groups + of % padded // c["group"]
            y[m] += x[:, part].double() @ ((q - 8.0) * s[:, of])
    return y.reshape(rows, heads, padded)[:, :, :c["outputs"]]


def _cells(pattern):
    return torch.stack([(pattern >> i) & 1 for i in range(32)], -1).reshape(pattern.shape[0], -1)


def _exact_select(logits, scores, beams, live):
    """The definition in 64 bits: candidates in order of their scores as they are given back (float32), then of their place."""
    groups, into, outputs = logits.shape
    x = logits.double().clone()
    if live is not None:
        for g, n in enumerate(live.tolist()):
            x[g, :, n:] = -math.inf
    p = scores.double()[:, :, None] + torch.log_softmax(x, -1)
    p = torch.where(p.isnan(), torch.full_like(p, -math.inf), p).reshape(groups, -1)
    at = p.float().sort(dim=1, descending=True, stable=True).indices[:, :beams]
    best = p.gather(1, at)
    gone = best == -math.inf
    slot = torch.arange(at.shape[1], device="cuda").clamp(max=into - 1).expand_as(at)
    parent, bucket = torch.where(gone, slot, at // outputs), torch.where(gone, -1, at % outputs)
    more = beams - at.shape[1]  # fewer candidates than beams
    if more > 0:
        best = torch.cat((best, best.new_full((groups, more), -math.inf)), 1)
        slot = torch.arange(at.shape[1], beams, device="cuda").clamp(max=into - 1).expand(groups, more)
        parent, bucket = torch.cat((parent, slot), 1), torch.cat((bucket, bucket.new_full((groups, more), -1)), 1)
    return best, parent.int(), bucket.int()


def _exact_reorder(states, parent):
    groups, beams = parent.shape
    rows = torch.arange(groups, device="cuda").repeat_interleave(beams) * beams + parent.reshape(-1)
    return [t.index_select(0, rows) for t in states]


def exact(case, seed):
    s, c, kind = prepare(case, seed), case, case["kind"]
    if kind == "logits":
        return _exact_logits(c, s["records"], _cells(s["pattern"]))
    if kind == "probabilities":
        y = _exact_logits(c, s["records"], _cells(s["pattern"]))
        out = torch.zeros_like(y)
        for row in range(y.shape[0]):
            n = int(s["live"][row // (y.shape[0] // c["models"])])
            out[row, :, :n] = torch.softmax(y[row, :, :n], -1)
        return out
    if kind == "matvec":
        return _exact_logits(c, s["records"], s["x"])
    if kind == "select":
        return _exact_select(s["logits"], s["scores"], c["beams"], s["live"])
    if kind == "reorder":
        return _exact_reorder(s["states"], s["parent"])
    scores, parent, bucket = _exact_select(s["logits"], s["scores"], c["beams"], None)
    return scores, parent, bucket, _exact_reorder(s["states"], parent)


# ---------------------------------------------------------------- work
def _row_bytes(cells, columns):
    return 4 * cells // 8 + 4 * columns + 2 * HISTORY * ACTIVE + HEADER


def _mean_active(inputs, columns):
    """Cells set in one pattern, on average."""
    n = min(40, columns)
    return 0.4 * n * (inputs // columns) + 0.6 * (n + 110)


def work(case):
    c, kind = case, case["kind"]
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    bytes_, flops = 0, 0
    if kind in ("logits", "probabilities"):
        rows, heads, models = c["rows"], c["heads"], c["models"]
        padded, groups, codes, _ = _layout(c)
        active = _mean_active(c["inputs"], _columns(c))
        # inputs of a matrix that any of its rows reads: each is read once
        read = c["inputs"] * (1 - (1 - active / c["inputs"]) ** (rows // models))
        bytes_ += models * read * (codes + 2 * heads * groups) + rows * c["inputs"] // 8
        bytes_ += 4 * rows * heads * c["outputs"]
        flops += 2 * rows * active * heads * c["outputs"]
    if kind == "matvec":
        padded, groups, codes, _ = _layout(c)
        read = c["inputs"] * (1 - (1 - c["filled"]) ** c["rows"])
        bytes_ += read * (codes + 2 * c["heads"] * groups) + c["rows"] * c["inputs"] * size[c["dtype"]]
        bytes_ += 4 * c["rows"] * c["heads"] * c["outputs"]
        flops += 2 * c["rows"] * c["filled"] * c["inputs"] * c["heads"] * c["outputs"]
    if kind == "select":
        bytes_ += c["groups"] * (c["beams_in"] * (size[c["dtype"]] * c["outputs"] + 4) + 12 * c["beams"])
        flops += 4 * c["groups"] * c["beams_in"] * c["outputs"]
    if kind == "step":
        bytes_ += c["groups"] * c["beams"] * (4 * c["outputs"] + 16)
        flops += 4 * c["groups"] * c["beams"] * c["outputs"]
    if kind in ("reorder", "step"):
        b = c["beams"]
        # parents drawn by the square of an even number: so many of the b have a child
        parents = sum(1 - (1 - (math.sqrt((k + 1) / b) - math.sqrt(k / b))) ** b for k in range(b))
        bytes_ += c["groups"] * (b + parents) * _row_bytes(c["cells"], c["columns"])
    return {"bytes": bytes_, "flops": flops}
