"""Batched counterparts of the reference's drivers.

* `SLOHarness` -- ModelTesting.py's SLO-violation prediction (runModel
  :36-107, processpredictionList :113-146, getModelStats :148-171) for N
  streams at once, on the GPU (csrc/slo.hip through the C ABI).
* `model_training` / `model_testing` -- the record loops of ModelTraining.py
  (:21-56, :80-97) and ModelTesting.py (:36-107, :194-213) for Model 1, over
  [records, streams] value arrays: record skipping on missing metrics, the
  save of network1 BEFORE the 2185th record's step (NetworkModel.py:123-127),
  TM learning switched off on the first test record while the SP keeps
  learning (NetworkModel.py:40-44), and 1 + 7 network steps per test record
  fed the same value (ModelTesting.py:66-72).
* `model_forecast` -- a look-ahead that feeds its own predictions instead:
  beams of bucket sequences per stream over the fleets of one model.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from ._lib import check

ANOMALY_SCORE = 0.85      # ModelTesting.py:30 (the README's sweep uses 0.98 / 0.99)
MAX_LEAD_TIME = 50        # ModelTesting.py:31
SLO_RESPONSE_TIME = 70    # ModelTesting.py:32
SAVE_FREQUENCY = 2185     # NetworkUtils.py:67
LOOKAHEAD = 7             # len(results[0]) of NetworkModel.py:19-20


class SLOHarness:
    """Per-stream SLO prediction state machine on the GPU."""

    def __init__(self, n_streams: int, threshold: float = ANOMALY_SCORE, max_lead: int = MAX_LEAD_TIME,
                 slo_response: int = SLO_RESPONSE_TIME, device: int | None = None):
        import torch
        self._L = _lib.lib()
        self.n_streams = int(n_streams)
        self.device = torch.cuda.current_device() if device is None else int(device)
        h = ctypes.c_void_p()
        check(self._L.htm_slo_create(self.n_streams, float(threshold), int(max_lead), int(slo_response),
                                     self.device, ctypes.byref(h)))
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            self._L.htm_slo_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _dev(self, x, dtype):
        import torch
        t = x if isinstance(x, torch.Tensor) else torch.as_tensor(np.asarray(x))
        t = t.to(device=f"cuda:{self.device}", dtype=dtype).contiguous()
        if t.numel() != self.n_streams:
            raise ValueError("expected one value per stream")
        return t

    def record(self, window_scores, violations, means, valid=None):
        """One runModel record of every stream: window_scores [w, n_streams]
        float32 device tensor (the engine's scores of the record's 1 + 7
        steps), violations / int(mean) per stream, valid = False skips the
        stream's record (a null cpu/mem, :51-53)."""
        import torch
        w = window_scores
        if not isinstance(w, torch.Tensor) or w.dtype != torch.float32 or w.dim() != 2 or \
                w.shape[1] != self.n_streams:
            raise ValueError("window_scores must be a float32 [window, n_streams] tensor")
        w = w.to(f"cuda:{self.device}").contiguous()
        v = self._dev(violations, torch.int32)
        m = self._dev(means, torch.int32)
        ok = self._dev(valid, torch.uint8) if valid is not None else None
        st = ctypes.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)
        check(self._L.htm_slo_record(self.h, ctypes.c_void_p(w.data_ptr()), int(w.shape[0]),
                                     ctypes.c_void_p(v.data_ptr()), ctypes.c_void_p(m.data_ptr()),
                                     ctypes.c_void_p(ok.data_ptr()) if ok is not None else None, st))
        self._keep = (w, v, m, ok)  # alive until the kernel has read them

    def stats(self) -> np.ndarray:
        """getModelStats per stream: int64 [n_streams, 5] = TP, FP, TN, FN, lead-time sum."""
        import torch
        out = np.zeros((self.n_streams, 5), np.int64)
        st = ctypes.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)
        check(self._L.htm_slo_stats(self.h, out.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)), st))
        return out


class AnomalyLikelihood:
    """NuPIC's AnomalyLikelihood.anomalyProbability for N streams at once on
    the GPU (csrc/likelihood.hip; parity unpinned -- the reference has no
    likelihood).  Defaults are NuPIC's."""

    def __init__(self, n_streams: int, learning_period: int = 288, estimation_samples: int = 100,
                 historic_window: int = 8640, reestimation_period: int = 100, device: int | None = None):
        import torch
        self._L = _lib.lib()
        self.n_streams = int(n_streams)
        self.device = torch.cuda.current_device() if device is None else int(device)
        h = ctypes.c_void_p()
        check(self._L.htm_likelihood_create(self.n_streams, int(learning_period), int(estimation_samples),
                                            int(historic_window), int(reestimation_period), self.device,
                                            ctypes.byref(h)))
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            self._L.htm_likelihood_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def anomaly_probability(self, values, scores, out=None):
        """values: device float64 [n_streams] or [n_streams, fields] (field 0 is
        the metric); scores: device float32 [n_streams].  Returns float64 [n]."""
        import torch
        v = values.contiguous()
        stride = 1 if v.dim() == 1 else v.shape[1]
        if v.dtype != torch.float64 or v.shape[0] != self.n_streams:
            raise ValueError("values must be float64 [n_streams(, fields)]")
        sc = scores.contiguous()
        if sc.dtype != torch.float32 or sc.numel() != self.n_streams:
            raise ValueError("scores must be float32 [n_streams]")
        if out is None:
            out = torch.empty(self.n_streams, dtype=torch.float64, device=sc.device)
        st = ctypes.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)
        check(self._L.htm_likelihood_step(self.h, ctypes.c_void_p(v.data_ptr()), int(stride),
                                          ctypes.c_void_p(sc.data_ptr()), ctypes.c_void_p(out.data_ptr()), st))
        return out


def valid_records(cpu, mem):
    """ModelTraining.py:29-32 / ModelTesting.py:51-53: a record with a null cpu
    or mem is skipped."""
    return ~(np.isnan(np.asarray(cpu, np.float64)) | np.isnan(np.asarray(mem, np.float64)))


def model_training(engine, cpu, save_path=None):
    """ModelTraining.runModel over cpu[records] (one stream: [records]; N
    streams sharing the record sequence: [records, N]).  Every stream sees
    every valid record once with SP and TM learning on; when the record
    counter reaches SAVE_FREQUENCY the engine is saved BEFORE that record's
    step (NetworkModel.py:123-127).  Returns the scores [steps, N]."""
    import torch
    v = np.asarray(cpu, np.float64)
    v = v.reshape(v.shape[0], -1)
    engine.set_learning(True, True)
    dev = f"cuda:{engine.device}"
    vals = torch.tensor(v, device=dev)
    n = v.shape[0]
    out = torch.empty((n, engine.n_streams), dtype=torch.float32, device=dev)
    k_save = SAVE_FREQUENCY - 1 if (save_path and n >= SAVE_FREQUENCY) else n
    engine.run(vals[:k_save], out=out[:k_save])
    engine.status()  # raise on pool / queue overflow (NuPIC's NTA_THROW)
    if k_save < n:
        engine.save(save_path)
        engine.run(vals[k_save:], out=out[k_save:])
        engine.status()
    return out


def model_testing(engine, cpu, violations, means, threshold=ANOMALY_SCORE, lookahead=LOOKAHEAD, slo=None,
                  chunk_records=256):
    """ModelTesting.runModel over test records for every stream: TM learning
    off (SP learning on), 1 + lookahead steps per record fed the record's
    value, the scores judged by the SLO harness on the GPU.  cpu / violations
    / means: [records] or [records, N].  Returns (windows [records, 1 +
    lookahead, N] float32 on the host, stats int64 [N, 5])."""
    import torch
    v = np.asarray(cpu, np.float64)
    v = v.reshape(v.shape[0], -1)
    n_rec, n = v.shape
    if n != engine.n_streams:
        v = np.broadcast_to(v, (n_rec, engine.n_streams))
        n = engine.n_streams
    viol = np.broadcast_to(np.asarray(violations, np.int64).reshape(n_rec, -1), (n_rec, n)).astype(np.int32)
    mean = np.broadcast_to(np.asarray(means).reshape(n_rec, -1), (n_rec, n)).astype(np.float64).astype(np.int32)
    w = 1 + lookahead
    slo = slo if slo is not None else SLOHarness(n, threshold=threshold, device=engine.device)
    engine.set_learning(True, False)  # NetworkModel.py:40-44 on the first test record
    dev = f"cuda:{engine.device}"
    windows = np.zeros((n_rec, w, n), np.float32)
    for r0 in range(0, n_rec, chunk_records):
        m = min(chunk_records, n_rec - r0)
        steps = torch.tensor(np.repeat(v[r0:r0 + m], w, axis=0), device=dev)  # [m * w, n]
        sc = engine.run(steps)
        vv = torch.tensor(viol[r0:r0 + m], device=dev)
        mm = torch.tensor(mean[r0:r0 + m], device=dev)
        for j in range(m):
            slo.record(sc[j * w:(j + 1) * w], vv[j], mm[j])
        windows[r0:r0 + m] = sc.reshape(m, w, n).cpu().numpy()
        engine.status()  # raise on pool / queue overflow (NuPIC's NTA_THROW)
    return windows, slo.stats()


def model_forecast(fleet, beam_fleet, readout, cpu, horizon=LOOKAHEAD, bucket_values=None, source="tm_output"):
    """The next `horizon` values of every stream after each record.

    The reference steps its network seven more times per record with the
    record's own value (ModelTesting.py:66-72) and reads the classifier's seven
    heads apart (NetworkUtils.py:166-184).  Here the network is fed what it
    predicts: after a record's step every stream forks into `beams` copies;
    each look-ahead step scores all (beam, bucket) continuations with the
    one-step read-out, keeps the best `beams`, lets their states go on from
    their parents' and feeds each its bucket's value.

    fleet: HTMEngine.fleet of G streams; beam_fleet: one of G * beams streams
    (beams <= 64) of the same model; readout: a Readout4 with one head, one
    matrix or one a stream; cpu: [records] or [records, G].  bucket_values:
    float64 [n_outputs], the value fed for each bucket (default: the scalar
    encoder's bucket centres).  source: "tm_output" (cells) or
    "col_confidence" (columns), what the read-out reads.

    Returns dict(values float64 [records, horizon, G], the best beam's; logp
    float32 [records, G], its log-probability; scores float32 [records, G], the
    records' anomaly scores), on the host.  Streams whose read-out leaves no
    bucket forecast NaN."""
    import torch
    from .beam import beam_reorder, beam_select
    g = fleet.n_streams
    if not fleet.is_fleet or not beam_fleet.is_fleet or beam_fleet.n_streams % g or beam_fleet is fleet:
        raise ValueError("model_forecast needs two fleets of one model, of G and of G * beams streams")
    if beam_fleet.n_streams // g > 64:
        raise ValueError("at most 64 beams (got %d)" % (beam_fleet.n_streams // g))
    if fleet.n_fields != 1:
        raise ValueError("model_forecast follows one encoder field (got %d)" % fleet.n_fields)
    beams, horizon = beam_fleet.n_streams // g, int(horizon)
    if horizon < 1:
        raise ValueError("horizon must be >= 1")
    if readout.n_heads != 1 or readout.n_models not in (1, g):
        raise ValueError("the read-out must have one head and one matrix, or one for each of the %d streams" % g)
    if source not in ("tm_output", "col_confidence"):
        raise ValueError("source must be 'tm_output' or 'col_confidence'")
    width = fleet.n_cells if source == "tm_output" else fleet.n_columns
    if readout.n_inputs != width:
        raise ValueError("the read-out has %d inputs, %s %d" % (readout.n_inputs, source, width))
    if beam_fleet.device != fleet.device or readout.device != torch.device("cuda", fleet.device):
        raise ValueError("the fleets and the read-out must be on one device")
    if beam_fleet.model_id() != fleet.model_id():
        raise ValueError("model_forecast needs two fleets of one model: these were built from different ones")
    dev = f"cuda:{fleet.device}"
    c = fleet.config
    if bucket_values is None:
        if c.enc_type != _lib.ENC_SCALAR or readout.n_outputs > c.enc_n - c.enc_w + 1:
            raise ValueError("give bucket_values: the read-out's outputs are not the scalar encoder's buckets")
        lo, hi = (c.field_minval[0], c.field_maxval[0]) if c.field_maxval[0] > c.field_minval[0] else (c.enc_minval, c.enc_maxval)
        bucket_values = lo + np.arange(readout.n_outputs) * ((hi - lo) / (c.enc_n - c.enc_w))
    table = torch.as_tensor(bucket_values, dtype=torch.float64, device=dev).reshape(-1)
    if table.numel() != readout.n_outputs:
        raise ValueError("bucket_values needs one value per output (%d)" % readout.n_outputs)
    table = torch.cat((table, table.new_full((1,), float("nan"))))  # [-1]: no bucket, a missing value
    v = np.asarray(cpu, np.float64)
    v = v[:, None] if v.ndim < 2 else v
    v = torch.tensor(np.ascontiguousarray(np.broadcast_to(v, (v.shape[0], g))), device=dev)
    n = v.shape[0]
    live = None
    if readout.live is not None:
        live = readout.live if readout.n_models == g else readout.live.expand(g)
    fork = torch.arange(g, dtype=torch.int32, device=dev).repeat_interleave(beams)
    start = torch.zeros((g, 1), dtype=torch.float32, device=dev)
    values = torch.empty((n, horizon, g), dtype=torch.float64, device=dev)
    logp = torch.empty((n, g), dtype=torch.float32, device=dev)
    scores = torch.empty((n, g), dtype=torch.float32, device=dev)
    path = torch.empty((g, beams, horizon), dtype=torch.int32, device=dev)

    def answer(eng, k):
        x = eng.get_output(source)
        y = readout.logits(x) if source == "tm_output" else readout.matvec(x)
        return y.view(g, k, readout.n_outputs)

    for t in range(n):
        fleet.step(v[t], out=scores[t])
        total, _, bucket = beam_select(answer(fleet, 1), start, beams, live=live)
        path[:, :, 0] = bucket
        for h in range(1, horizon):
            if h == 1:
                beam_fleet.copy_streams(fleet, fork)
            beam_fleet.step(table[bucket.reshape(-1).long()])
            total, parent, bucket = beam_select(answer(beam_fleet, beams), total, beams, live=live)
            beam_reorder([path], parent)
            path[:, :, h] = bucket
            if h + 1 < horizon:
                beam_fleet.reorder_streams(parent)
        values[t] = table[path[:, 0].long()].t()
        logp[t] = total[:, 0]
    fleet.status()  # raise on pool / queue overflow (NuPIC's NTA_THROW)
    beam_fleet.status()
    return dict(values=values.cpu().numpy(), logp=logp.cpu().numpy(), scores=scores.cpu().numpy())
