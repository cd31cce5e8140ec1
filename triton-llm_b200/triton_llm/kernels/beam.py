"""Beam search on the device: selection over beams and vocabulary, and the
reordering of the beams' page tables (the reference selects greedily or by
sampling, smollm2_triton/model.py:566-584).

Tensors and streams as in ``triton_llm.kernels.paged``.
"""

from __future__ import annotations

import ctypes
import math

from triton_llm import gpu, _lib
from ._common import device_of, dtype_code, on_device, require_gpu, strides
from .paged import _workspace


class BeamWorkspace:
    """Scratch of ``beam_select`` (allocated once; calls that overlap on the
    GPU need one each). Ready for any stream when it has been made, and released
    only after the device's work."""

    def __init__(self, groups, beams, vocab, k):
        n = ctypes.c_size_t()
        _lib.call("tllm_beam_workspace", int(groups), int(beams), int(vocab), int(k),
                  ctypes.byref(n))
        self._buf = gpu.Scratch(n.value)
        self.ptr, self.nbytes = self._buf.data_ptr(), n.value


def beam_select(logits, scores, out_scores, out_parents, out_tokens, done=None,
                pad_token=0, out_done=None, eos_token=-1, workspace=None, stream=None):
    """The k best continuations of every group of beams.

    logits   (groups * beams, vocab) float32, rows contiguous
    scores   (groups, beams) float32: the beams' log-probabilities (-inf: none)
    out_scores, out_parents, out_tokens
             (groups, k) float32 / int32 / int32, best first: the candidate's
             score ``scores[b] + log_softmax(logits[b])[t]``, its beam b within
             the group and its token t; equal scores by the lower beam, within
             a beam by the larger logit, then the lower token; k <= 64
    done     (groups, beams) or (groups * beams,) int32 or None: a beam with a
             value != 0 has one candidate, ``pad_token`` at its own score
    out_done (groups, k) int32 or None: whether the candidate's beam is done or
             its token is ``eos_token``
    """
    shape, rows = scores.shape, logits.shape
    if len(shape) != 2 or len(rows) != 2:
        raise ValueError(f"scores and logits must be 2D, got {tuple(shape)}, {tuple(rows)}")
    groups, beams = shape
    n, vocab = rows
    if n != groups * beams:
        raise ValueError(f"logits have {n} rows, {groups} groups of {beams} beams")
    if dtype_code(logits, "logits") != _lib.F32:
        raise ValueError(f"logits must be float32, got {logits.dtype}")
    ld, one = strides(logits)
    if one != 1 and vocab > 1:
        raise ValueError("rows of logits must be contiguous")
    require_gpu(logits, "logits")
    out = out_scores.shape
    if len(out) != 2 or out[0] != groups:
        raise ValueError(f"out_scores must be ({groups}, k), got {tuple(out)}")
    k = out[1]
    flags = 0
    if done is not None:
        flags = on_device(done, "done", _lib.I32)
        if done.shape != shape and math.prod(done.shape) != n:
            raise ValueError(f"done has {math.prod(done.shape)} values for {n} beams")
    if workspace is None:
        if stream is not None:
            raise ValueError("a call on another stream needs its own workspace")
        # (one of a larger call holds a smaller one's parts; k > 64 is refused)
        rows = 1 << (n - 1).bit_length()
        most = 1 << (k - 1).bit_length() if k <= 64 else k
        workspace = _workspace(lambda: BeamWorkspace(rows, 1, max(vocab, most), most),
                               "beam", device_of(logits), rows, most)
    _lib.call("tllm_beam_select", _lib.BEAM_STEP.pack(
        logits.data_ptr(), on_device(scores, "scores", _lib.F32), flags,
        on_device(out_scores, "out_scores", _lib.F32),
        on_device(out_parents, "out_parents", _lib.I32, out),
        on_device(out_tokens, "out_tokens", _lib.I32, out),
        0 if out_done is None else on_device(out_done, "out_done", _lib.I32, out),
        workspace.ptr, workspace.nbytes, ld if n > 1 else 0, groups, beams, vocab, k,
        int(pad_token), int(eos_token)), stream)


def beam_reorder(parents, lens, table, table_out, copy_src, copy_dst, copy_fill, *,
                 page_size, stream=None):
    """Page tables after a selection step (``tllm_beam_reorder``).

    parents  (groups, beams) int32: the beam that each beam continues
    lens     (groups * beams,) int32: cached tokens before the step, equal
             within a group
    table    (groups * beams, pages) int32; table_out the same shape, or the
             same tensor to reorder in place
    copy_src, copy_dst, copy_fill
             (groups * beams,) int32: the page copies (``page_copy``) that the
             step needs; none where src == dst or src < 0
    Every beam has to own the page that it is filling and those after it.
    """
    shape, rows = parents.shape, table.shape
    if len(shape) != 2 or len(rows) != 2:
        raise ValueError(f"parents and table must be 2D, got {tuple(shape)}, {tuple(rows)}")
    groups, beams = shape
    n = groups * beams
    if rows[0] != n:
        raise ValueError(f"table has {rows[0]} rows for {n} beams")
    _lib.call("tllm_beam_reorder", _lib.BEAM_TABLES.pack(
        on_device(parents, "parents", _lib.I32), on_device(lens, "lens", _lib.I32, (n,)),
        on_device(table, "table", _lib.I32),
        on_device(table_out, "table_out", _lib.I32, rows),
        on_device(copy_src, "copy_src", _lib.I32, (n,)),
        on_device(copy_dst, "copy_dst", _lib.I32, (n,)),
        on_device(copy_fill, "copy_fill", _lib.I32, (n,)), groups, beams, rows[1],
        int(page_size)), stream)
