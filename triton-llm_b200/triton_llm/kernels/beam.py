"""Beam search on the device: selection over beams and vocabulary, and the
reordering of the beams' page tables (the reference selects greedily or by
sampling, smollm2_triton/model.py:566-584).

Tensors and streams as in ``triton_llm.kernels.paged``.
"""

from __future__ import annotations

import ctypes

import numpy as np

from triton_llm import gpu, _lib
from ._common import dtype_code, on_device, require_gpu, strides
from .paged import _workspace


class BeamWorkspace:
    """Scratch of ``beam_select`` (allocated once; calls that overlap on the
    GPU need one each)."""

    def __init__(self, groups, beams, vocab, k):
        n = ctypes.c_size_t()
        _lib.call("tllm_beam_workspace", int(groups), int(beams), int(vocab), int(k),
                  ctypes.byref(n))
        self._buf = gpu.zeros((max(n.value // 4, 1),), np.int32)
        self.ptr, self.nbytes = self._buf.data_ptr(), n.value


def beam_select(logits, scores, out_scores, out_parents, out_tokens, done=None,
                pad_token=0, out_done=None, eos_token=-1, workspace=None, stream=None):
    """The k best continuations of every group of beams.

    logits   (groups * beams, vocab) float32, rows contiguous
    scores   (groups, beams) float32: the beams' log-probabilities (-inf: none)
    out_scores, out_parents, out_tokens
             (groups, k) float32 / int32 / int32, best first: the candidate's
             score ``scores[b] + log_softmax(logits[b])[t]``, its beam b within
             the group and its token t; equal scores by the lower beam, then
             the lower token; k <= 64
    done     (groups, beams) or (groups * beams,) int32 or None: a beam with a
             value != 0 has one candidate, ``pad_token`` at its own score
    out_done (groups, k) int32 or None: whether the candidate's beam is done or
             its token is ``eos_token``
    """
    if len(scores.shape) != 2 or len(logits.shape) != 2:
        raise ValueError(f"scores and logits must be 2D, got {tuple(scores.shape)}, "
                         f"{tuple(logits.shape)}")
    groups, beams = int(scores.shape[0]), int(scores.shape[1])
    if logits.shape[0] != groups * beams:
        raise ValueError(f"logits have {logits.shape[0]} rows, {groups} groups of {beams} "
                         "beams")
    if dtype_code(logits, "logits") != _lib.F32:
        raise ValueError(f"logits must be float32, got {logits.dtype}")
    sl = strides(logits)
    vocab = int(logits.shape[1])
    if sl[1] != 1 and vocab > 1:
        raise ValueError("rows of logits must be contiguous")
    require_gpu(logits, "logits")
    if len(out_scores.shape) != 2 or out_scores.shape[0] != groups:
        raise ValueError(f"out_scores must be ({groups}, k), got {tuple(out_scores.shape)}")
    shape = tuple(out_scores.shape)
    k = int(shape[1])
    flags = None
    if done is not None:
        flags = on_device(done, "done", _lib.I32)
        n = 1
        for s in done.shape:
            n *= int(s)
        if n != groups * beams:
            raise ValueError(f"done has {n} values for {groups * beams} beams")
    args = (on_device(scores, "scores", _lib.F32),
            on_device(out_scores, "out_scores", _lib.F32),
            on_device(out_parents, "out_parents", _lib.I32, shape),
            on_device(out_tokens, "out_tokens", _lib.I32, shape))
    if workspace is None:
        if stream is not None:
            raise ValueError("a call on another stream needs its own workspace")
        workspace = _workspace(lambda: BeamWorkspace(groups, beams, vocab, k), "beam",
                               gpu.current_device(), groups, beams, vocab, k)
    _lib.call("tllm_beam_select", logits.data_ptr(), sl[0] if groups * beams > 1 else 0,
              args[0], flags, int(pad_token), groups, beams, vocab, k, args[1], args[2],
              args[3], int(eos_token),
              None if out_done is None else on_device(out_done, "out_done", _lib.I32, shape),
              workspace.ptr, workspace.nbytes, stream)


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
    if len(parents.shape) != 2 or len(table.shape) != 2:
        raise ValueError(f"parents and table must be 2D, got {tuple(parents.shape)}, "
                         f"{tuple(table.shape)}")
    groups, beams = int(parents.shape[0]), int(parents.shape[1])
    n = groups * beams
    if table.shape[0] != n:
        raise ValueError(f"table has {table.shape[0]} rows for {n} beams")
    shape = tuple(table.shape)
    _lib.call("tllm_beam_reorder", on_device(parents, "parents", _lib.I32),
              on_device(lens, "lens", _lib.I32, (n,)), on_device(table, "table", _lib.I32),
              on_device(table_out, "table_out", _lib.I32, shape), groups, beams,
              int(shape[1]), int(page_size),
              on_device(copy_src, "copy_src", _lib.I32, (n,)),
              on_device(copy_dst, "copy_dst", _lib.I32, (n,)),
              on_device(copy_fill, "copy_fill", _lib.I32, (n,)), stream)
