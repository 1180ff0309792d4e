"""Beam selection over beams x buckets, and the beams' states reordered.

The reference's look-ahead feeds the record's own value seven times
(ML/HTM/ModelTesting.py:66-72).  A forecast that feeds its predictions instead
(`harness.model_forecast`) follows several continuations of every stream: each
look-ahead step scores every (beam, next bucket), keeps the best, and lets the
kept beams' states go on from their parents'.  Kernels: csrc/beam.hip.
"""
from __future__ import annotations

import array

from . import _lib
from ._lib import check
from .readout import _On, dtype_code

MAX_BEAMS = 64
MAX_BUFFERS = 32
MAX_GROUPS = 2 ** 31 - 1
_WHOLE = None  # dtypes of whole numbers and bits: never a view still to be conjugated or negated


def beam_select(logits, scores, beams: int, live=None):
    """The `beams` best of each group's beams_in x n_outputs continuations.

    logits [groups, beams_in, n_outputs] float32 / float16 / bfloat16 (any
    strides whose last is 1; others are copied); scores float32 [groups,
    beams_in], the beams' summed log-probabilities so far; live: optional
    int32 [groups], how many outputs are in use.  A continuation's score is

        float32((logits[w, o] - m) + (scores[w] - log(sum_{o' < live} exp(logits[w, o'] - m))))

    in float64 up to that one rounding, m the beam's largest live logit.  Returns (scores float32,
    parent int32, output int32), each [groups, beams], best first, equal scores
    by the lower (parent, output).  Continuations of score -inf or NaN are
    never taken: a slot left over has score -inf, output -1 and parent
    min(slot, beams_in - 1)."""
    import torch
    L = _lib.lib()
    code = dtype_code(logits.dtype) if isinstance(logits, torch.Tensor) else -1
    if code not in (0, 2, 3) or logits.dim() != 3 or not logits.is_cuda:
        raise ValueError("logits must be a float32, float16 or bfloat16 CUDA tensor [groups, beams_in, n_outputs]")
    groups, win, v = logits.shape
    dev = logits.device
    beams = int(beams)
    if not 1 <= win <= MAX_BEAMS or not 1 <= beams <= MAX_BEAMS or v < 1 or win * v > 2 ** 30:
        raise ValueError("1..%d beams in and out, n_outputs >= 1 and beams_in * n_outputs <= 2**30 (got %d, %d, %d)" %
                         (MAX_BEAMS, win, beams, v))
    if groups > MAX_GROUPS:
        raise ValueError("at most 2**31 - 1 groups (got %d)" % groups)
    if not isinstance(scores, torch.Tensor) or scores.dtype != torch.float32 or scores.device != dev or \
            scores.shape != (groups, win):
        raise ValueError("scores must be float32 [groups, beams_in] on %s" % dev)
    if (logits.requires_grad or scores.requires_grad) and torch.is_grad_enabled():
        raise ValueError("a selection has no gradient: detach the logits and scores")
    if live is not None and (not isinstance(live, torch.Tensor) or live.dtype != torch.int32 or live.device != dev or
                             live.shape != (groups,)):
        raise ValueError("live must be int32 [groups] on %s" % dev)
    logits = logits.resolve_neg()
    gs, bs, vs = logits.stride()
    if vs != 1 and v > 1:
        logits = logits.contiguous()
        gs, bs, _ = logits.stride()
    scores = scores.resolve_neg().contiguous()
    live = live.contiguous() if live is not None else None
    with _On(dev.index) as stream:
        o_score, o_parent, o_bucket = scores.new_empty((3, groups, beams), dtype=torch.int32).unbind(0)
        o_score = o_score.view(torch.float32)
        nb = L.htm_beam_work_bytes(groups, win, beams, v)
        work = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        check(L.htm_beam_select(logits.data_ptr(), code, gs, bs, scores.data_ptr(),
                                live.data_ptr() if live is not None else None, groups, win, beams, v,
                                o_score.data_ptr(), o_parent.data_ptr(), o_bucket.data_ptr(),
                                work.data_ptr() if nb else None, nb, stream))
    return o_score, o_parent, o_bucket


def beam_reorder(buffers, parent, out=None):
    """Row (g, w) of every buffer becomes row (g, parent[g, w]).

    buffers: up to 32 contiguous CUDA tensors of any type, [groups * beams, ...]
    or [groups, beams, ...]; parent: int32 [groups, beams] (a parent outside
    0..beams-1 counts as w itself).  out: tensors like the buffers to write to;
    None reorders in place, and a buffer that stands in `out` as well is
    reordered in place.  Buffers that overlap otherwise are refused, and so are
    those that require a gradient.  Returns the reordered tensors as a list."""
    import torch
    global _WHOLE
    if _WHOLE is None:
        _WHOLE = {torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.bool}
    L = _lib.lib()
    buffers = list(buffers)
    dst = buffers if out is None else list(out)
    if not isinstance(parent, torch.Tensor) or parent.dtype != torch.int32 or parent.dim() != 2 or \
            not parent.is_cuda or not 1 <= parent.shape[1] <= MAX_BEAMS:
        raise ValueError("parent must be an int32 CUDA tensor [groups, 1..%d beams]" % MAX_BEAMS)
    if not 1 <= len(buffers) <= MAX_BUFFERS or len(dst) != len(buffers):
        raise ValueError("1..%d buffers and as many destinations" % MAX_BUFFERS)
    groups, beams = parent.shape
    if groups > MAX_GROUPS:
        raise ValueError("at most 2**31 - 1 groups (got %d)" % groups)
    rows = groups * beams
    dev = parent.device
    parent = parent.contiguous()
    n = len(buffers)
    p = [0] * (3 * n)  # sources, destinations, row bytes
    grad = False
    index, tensor = dev.index, torch.Tensor
    for k, a in enumerate(buffers):
        b = dst[k]
        ok = isinstance(a, tensor) and a.get_device() == index and a.is_contiguous()
        if ok:
            shape = a.shape
            grad = grad or a.requires_grad
        if ok and b is not a:
            ok = isinstance(b, tensor) and b.get_device() == index and b.dtype is a.dtype and b.shape == shape and b.is_contiguous()
            if ok:
                grad = grad or b.requires_grad
                ok = a.dtype in _WHOLE or a.is_conj() == b.is_conj() and a.is_neg() == b.is_neg()
        if not ok:
            raise ValueError("buffers and destinations must be contiguous, alike, and on %s" % dev)
        if not shape or shape[0] != rows and shape[:2] != (groups, beams):
            raise ValueError("a buffer must be [groups * beams, ...] or [groups, beams, ...] for %d groups of %d, got %s" %
                             (groups, beams, tuple(shape)))
        p[k], p[n + k], p[2 * n + k] = a.data_ptr(), b.data_ptr(), a.nbytes // rows if rows else 0
    if grad and torch.is_grad_enabled():
        raise ValueError("a reordering has no gradient: detach the buffers")
    p = array.array("Q", p)
    at = p.buffer_info()[0]
    with _On(dev.index) as stream:
        check(L.htm_beam_reorder(n, at, at + 8 * n, at + 16 * n, parent.data_ptr(), groups, beams, stream))
    torch._C._increment_version(dst)  # (a backward pass that has kept one of them notices)
    return dst
