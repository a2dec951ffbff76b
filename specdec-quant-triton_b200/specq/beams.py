"""Beam search's step on the device: the best continuations, and the beams' states moved to follow them.

    beam_select(logits, scores, n=None, done=None, pad=0)    -> (scores', parent, token)
    beam_reorder(states, parent)                              in place

parent holds row numbers, so it goes to `pages_fork` as it is, and the block-scaled cache follows the beams by
sharing pages; beam_reorder moves what stands beside the cache (token histories, lengths, recurrent
states).  Nothing is synchronised, and both may be captured in a CUDA graph.  There is no reference counterpart.
"""
from __future__ import annotations

from . import _lib

# The argument checks and the calls are in csrc/py_blocks.cpp.
_native = _lib.native()


def beam_select(logits, scores, n=None, done=None, pad=0, beams=None):
    """The n best continuations of each request (n = None: as many as it has beams).

    logits [R, V] float16, bfloat16 or float32 (any row stride): request b's beams are rows b * beams and on.
    scores float32 [B, beams] (or [R] with `beams` given): the beams' log-probabilities so far; -inf: an empty
    beam.  Candidate (row, token) has the total score + log_softmax(logits)[token].  done (bool, R): a finished
    beam goes on as itself only, by the token `pad` at its own score.

    Returns scores' float32, parent int32 (rows) and token int32, each [B, n], best first; equal totals (in 64
    bits) by beam, then token.  A beam's log-sum-exp is good to some 1e-7 (2e-6 at worst), so totals of different
    beams that are closer than that come in either order, those of equal rows too unless the rows begin alike
    (their addresses modulo 16 bytes); and so do logits of one beam too close for their totals in 64 bits.  A candidate of total -inf (a masked token) is never chosen: a place that is left
    without one has score -inf, token `pad` and the row b * beams + j % beams, which for j < beams is
    the place's own.  NaN logits count as -inf, +inf ones as their type's largest finite number; a NaN or +inf score as -inf.
    Up to 64 beams and n = 128."""
    return _native.beam_select(logits, scores, n, done, pad, beams)


def beam_reorder(states, parent, beams=None):
    """Row r of every tensor of `states` ([R, ...], rows contiguous, any type) becomes its row parent[r], as it was
    before the call: in place, all at once.  parent int32 [B, beams] (or [R] with `beams` given) has rows of
    the same request; a negative one keeps the row, and so does one of another request, which the
    status word reports.  States must not share memory.  Up to 64 beams."""
    _native.beam_reorder(states, parent, beams)
