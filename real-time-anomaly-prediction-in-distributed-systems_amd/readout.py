"""4-bit read-out of cells or columns: a frozen SDRClassifier's answer for
fleets.

The reference's Model 1 reads its classifier once learning is off
(ML/HTM/NetworkModel.py:40-44,70-97, ML/HTM/NetworkUtils.py:166-184).  The
classifier here keeps NuPIC's float64 matrices, 660 MB a Model-1 stream; a
`Readout4` holds the same weights in 4 bits with one bfloat16 scale per group
of neighbouring buckets (47 MB a stream, or 47 MB for a whole fleet that
shares its model) and computes

    y[r, h, o] = sum_i x[r, i] * scale[m, i, h, o // group] * (code[m, i, h, o] - 8)

with float32 sums in csrc/readout.hip (htm_q4_*).  Consecutive rows share a
matrix: row r of n reads model m = r // (n // n_models).
"""
from __future__ import annotations

import ctypes

from . import _lib
from ._lib import check

_DTYPES = None


def dtype_code(dtype) -> int:
    """HTM_T_* of a torch dtype, -1 for any other."""
    global _DTYPES
    if _DTYPES is None:
        import torch
        _DTYPES = {torch.float32: 0, torch.float64: 1, torch.float16: 2, torch.bfloat16: 3}
    return _DTYPES.get(dtype, -1)


class _On:
    """`with _On(index) as stream`: CUDA device `index` is current inside, `stream` its current stream's handle.
    (torch.cuda.device and current_stream cost some 4 us a call, half of a small launch's host time.)"""

    __slots__ = ("index", "before")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        import torch
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch._C._cuda_setDevice(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            import torch
            torch._C._cuda_setDevice(self.before)


def _q4_shape(*sizes):
    """The htm_q4_shape of (n_models, n_inputs, n_heads, n_outputs, group)."""
    for k in sizes:
        if not -2 ** 31 <= k < 2 ** 31:
            raise ValueError("a read-out's sizes are below 2**31 (got %s)" % (sizes,))
    return _lib.Q4Shape(*sizes)


class Readout4:
    """The 4-bit matrices of n_models read-outs, n_inputs x n_heads x
    n_outputs each (heads: the classifier's look-ahead steps).

    `records`: uint8 CUDA tensor [n_models, n_inputs, record bytes] in the
    layout of htm_q4_shape (include/htm_amd.h); `quantize`, `from_classifier`
    and `SDRClassifier.readout4` make it.  Its scales must be 0 or of a size
    within 2**-110 .. 2**100; others raise ValueError (the check waits for the
    device, and is left out while a graph is captured).  `live`: optional int32 [n_models],
    how many of a head's outputs are in use (`probabilities`' default)."""

    def __init__(self, records, n_inputs: int, n_heads: int, n_outputs: int, group: int = 32, live=None, *, _new=False):
        import torch
        self._L = _lib.lib()
        if not isinstance(records, torch.Tensor) or records.dtype != torch.uint8 or records.dim() != 3 or \
                not records.is_cuda or not records.is_contiguous():
            raise ValueError("records must be a contiguous uint8 CUDA tensor [n_models, n_inputs, record bytes]")
        self.n_models, self.n_inputs = int(records.shape[0]), int(n_inputs)
        self.n_heads, self.n_outputs, self.group = int(n_heads), int(n_outputs), int(group)
        self._shape = _q4_shape(self.n_models, self.n_inputs, self.n_heads, self.n_outputs, self.group)
        self._pshape = ctypes.addressof(self._shape)
        per = self._L.htm_q4_record_bytes(self._pshape)
        if not per:
            raise ValueError(self._L.htm_last_error().decode(errors="replace"))
        if records.shape[1] != self.n_inputs or records.shape[2] != per:
            raise ValueError("records must be [%d, %d, %d], got %s" %
                             (self.n_models, self.n_inputs, per, tuple(records.shape)))
        if records.data_ptr() % 16:
            raise ValueError("records must be 16-byte aligned")
        self.records = records
        self.device = records.device
        self._index = records.device.index
        self._rec = records.data_ptr()
        self.live = None if live is None else self._live(live)
        if not _new and not torch.cuda.is_current_stream_capturing():
            with _On(self._index) as stream:
                bad = torch.zeros(1, dtype=torch.int32, device=self.device)
                check(self._L.htm_q4_check(self._pshape, self._rec, bad.data_ptr(), stream))
                if bad.item():
                    raise ValueError("the records' scales must be 0 or of a size within 2**-110 .. 2**100")

    # ------------------------------------------------------------- making one
    @classmethod
    def record_bytes(cls, n_models: int, n_inputs: int, n_heads: int, n_outputs: int, group: int = 32) -> int:
        """Bytes of one input's record."""
        L = _lib.lib()
        s = _q4_shape(int(n_models), int(n_inputs), int(n_heads), int(n_outputs), int(group))
        per = L.htm_q4_record_bytes(ctypes.addressof(s))
        if not per:
            raise ValueError(L.htm_last_error().decode(errors="replace"))
        return per

    @classmethod
    def quantize(cls, weights, group: int = 32, live=None) -> "Readout4":
        """From float32 / float64 CUDA weights [n_models, n_inputs, n_heads,
        n_outputs].  Raises ValueError for infinite or NaN weights (this waits
        for the device)."""
        import torch
        if not isinstance(weights, torch.Tensor) or not weights.is_cuda or weights.dim() != 4 or \
                weights.dtype not in (torch.float32, torch.float64):
            raise ValueError("weights must be a float32 or float64 CUDA tensor [n_models, n_inputs, n_heads, n_outputs]")
        weights = weights.resolve_neg()
        w = weights if weights.stride(3) == 1 or weights.shape[3] == 1 else weights.contiguous()
        if min(w.stride()[:3]) < 0:
            w = w.contiguous()
        nm, ni, nh, no = (int(k) for k in w.shape)
        per = cls.record_bytes(nm, ni, nh, no, group)
        with _On(w.device.index) as stream:
            rec = torch.zeros((nm, ni, per), dtype=torch.uint8, device=w.device)
            bad = torch.zeros(1, dtype=torch.int32, device=w.device)
            self = cls(rec, ni, nh, no, group, live, _new=True)
            check(self._L.htm_q4_quantise(self._pshape, w.data_ptr(), dtype_code(w.dtype), w.stride(0), w.stride(1),
                                          w.stride(2), self._rec, bad.data_ptr(), stream))
            if bad.item():
                raise ValueError("weights must be finite (and at most 7 * 2**100)")
        return self

    @classmethod
    def from_classifier(cls, classifier, s0: int = 0, n: int | None = None, group: int = 32,
                        steps=None) -> "Readout4":
        """The present weights of an SDRClassifier's streams [s0, s0 + n), one
        matrix a stream, and its live bucket counts.  steps: neighbouring
        entries of the classifier's steps to take as heads (default: all).
        Later learning of the classifier does not reach the read-out."""
        import torch
        n = classifier.n_streams - s0 if n is None else int(n)
        if s0 < 0 or n < 1 or s0 + n > classifier.n_streams:
            raise ValueError("streams [%d, %d) are not the classifier's" % (s0, s0 + n))
        steps = classifier.steps if steps is None else [int(k) for k in steps]
        y0, nh = (classifier.steps.index(steps[0]) if steps and steps[0] in classifier.steps else -1), len(steps)
        if y0 < 0 or classifier.steps[y0:y0 + nh] != steps:
            raise ValueError("steps %s are not neighbours in the classifier's %s" % (steps, classifier.steps))
        dev = torch.device("cuda", classifier.device)
        per = cls.record_bytes(n, classifier.n_inputs, nh, classifier.n_buckets, group)
        with _On(dev.index) as stream:
            rec = torch.zeros((n, classifier.n_inputs, per), dtype=torch.uint8, device=dev)
            live = torch.empty(n, dtype=torch.int32, device=dev)
            bad = torch.zeros(1, dtype=torch.int32, device=dev)
            self = cls(rec, classifier.n_inputs, nh, classifier.n_buckets, group, live, _new=True)
            check(self._L.htm_cls_quantise(classifier.h, int(s0), y0, self._pshape, self._rec, live.data_ptr(),
                                           bad.data_ptr(), stream))
            if bad.item():
                raise ValueError("the classifier's weights are not finite")
        return self

    # ------------------------------------------------------------------ checks
    def _live(self, live):
        import torch
        if not isinstance(live, torch.Tensor) or live.dtype != torch.int32 or live.device != self.device or \
                live.shape != (self.n_models,) or not live.is_contiguous():
            raise ValueError("live must be a contiguous int32 tensor [n_models] on %s" % self.device)
        return live

    def _rows(self, x, width, what):
        """(tensor, rows, row stride): rows of `width` elements, neighbouring in memory."""
        if x.device != self.device:
            raise ValueError("%s is on %s, the read-out on %s" % (what, x.device, self.device))
        if x.dim() != 2 or x.shape[1] != width:
            raise ValueError("%s must be [rows, %d], got %s" % (what, width, tuple(x.shape)))
        n = x.shape[0]
        if n >= 2 ** 31:
            raise ValueError("too many rows: %d" % n)
        if n % self.n_models:
            raise ValueError("%d rows do not divide over %d models" % (n, self.n_models))
        x = x.resolve_neg()
        if (x.stride(1) != 1 and width > 1) or (n > 1 and x.stride(0) < width):
            x = x.contiguous()
        return x, n, x.stride(0)

    def _out(self, out, n, *reads):
        import torch
        shape = (n, self.n_heads, self.n_outputs)
        if out is None:
            return self.records.new_empty(shape, dtype=torch.float32)
        if not isinstance(out, torch.Tensor) or out.dtype != torch.float32 or out.device != self.device or \
                out.shape != shape or not out.is_contiguous() or out.is_neg():
            raise ValueError("out must be a contiguous float32 tensor %s on %s" % (shape, self.device))
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("a frozen read-out has no gradient: detach out")
        o0 = out.data_ptr()
        for t in (self.records, *reads):  # (a workgroup writes while others still read)
            if t is not None and t.numel():
                size = sum((k - 1) * s for k, s in zip(t.shape, t.stride())) + 1
                if t.data_ptr() < o0 + out.nbytes and o0 < t.data_ptr() + size * t.element_size():
                    raise ValueError("out overlaps what the call reads")
        torch._C._increment_version((out,))  # (a backward pass that has kept it notices)
        return out

    def _pattern(self, pattern):
        import torch
        if not isinstance(pattern, torch.Tensor) or pattern.dtype not in (torch.int32, torch.uint32):
            raise ValueError("patterns are int32 / uint32 word bitmaps [rows, n_inputs / 32]")
        if self.n_inputs % 32:
            raise ValueError("patterns need n_inputs a multiple of 32 (%d)" % self.n_inputs)
        return self._rows(pattern, self.n_inputs // 32, "the pattern")

    # --------------------------------------------------------------- products
    def logits(self, pattern, out=None):
        """y [rows, n_heads, n_outputs] float32 of word bitmaps [rows,
        n_inputs / 32] (the engine's "tm_output"): bit b of word w is input
        32 w + b.  A row without a set bit gives zeros.  out (of every product):
        a contiguous tensor to write to, apart from all that the call reads."""
        p, n, stride = self._pattern(pattern)
        y = self._out(out, n, p)
        with _On(self._index) as stream:
            check(self._L.htm_q4_logits(self._pshape, self._rec, p.data_ptr(), stride, n, y.data_ptr(), stream))
        return y

    def probabilities(self, pattern, live=None, out=None):
        """softmax of `logits` over each head's first `live` outputs (int32
        [n_models]; default: the read-out's own, or all of them), 0 above: the
        classifier region's "probabilities".  n_outputs <= 1024."""
        p, n, stride = self._pattern(pattern)
        lv = self.live if live is None else self._live(live)
        y = self._out(out, n, p, lv)
        with _On(self._index) as stream:
            check(self._L.htm_q4_probabilities(self._pshape, self._rec, p.data_ptr(), stride,
                                               lv.data_ptr() if lv is not None else None, n, y.data_ptr(), stream))
        return y

    def matvec(self, x, out=None):
        """y of vectors of numbers [rows, n_inputs], float32 / float16 /
        bfloat16 (the engine's "col_confidence", an averaged activity).  An
        infinite number makes its row's outputs infinite (NaN where the weight
        is zero), a NaN makes them NaN; other rows keep theirs.  With five and
        more rows a matrix, what lies below 2**-126 in a number's 8-bit parts,
        a product or a sum may count as zero."""
        import torch
        if not isinstance(x, torch.Tensor) or dtype_code(x.dtype) not in (0, 2, 3):
            raise ValueError("x must be a float32, float16 or bfloat16 tensor [rows, n_inputs]")
        if x.requires_grad and torch.is_grad_enabled():
            raise ValueError("a frozen read-out has no gradient: detach x")
        v, n, stride = self._rows(x, self.n_inputs, "x")
        y = self._out(out, n, v)
        nb = self._L.htm_q4_work_bytes(self._pshape, n)
        with _On(self._index) as stream:
            work = torch.empty(nb, dtype=torch.uint8, device=self.device) if nb else None
            check(self._L.htm_q4_matvec(self._pshape, self._rec, v.data_ptr(), dtype_code(v.dtype), stride, n,
                                        y.data_ptr(), work.data_ptr() if nb else None, nb, stream))
        return y

    def device_bytes(self) -> int:
        return self.records.numel()
