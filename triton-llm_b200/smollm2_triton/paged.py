"""Decoding over a paged KV cache: long and windowed contexts, forked sequences
and beam search (no counterpart in the reference, which keeps one preallocated
cache per sequence, smollm2_triton/model.py:219-225, and samples one
continuation, model.py:566-584).

``PagedSession`` is a ``LlamaSession`` whose caches are pages of one arena:

* a sequence takes pages as it grows, releases them when it ends and, with a
  sliding window, when they leave it;
* ``fork`` continues a sequence in another slot, sharing its full pages;
* ``compact`` moves the used pages together;
* a decode step projects q, k and v, rotates and appends them
  (``paged_append``), and attends over the pages (``paged_attention``); prompts
  run through the prefill kernels over one layer's staging cache, from which
  their keys and values are written into pages (``paged_write``).

``beam_search`` runs all of it with the selection over beams and vocabulary and
the reordering of the beams' pages on the device, one CUDA graph per step.
"""

from __future__ import annotations

import numpy as np

from triton_llm import gpu, _lib
from triton_llm.kernels import (BeamWorkspace, PagedKV, PagedWorkspace, beam_reorder,
                                beam_select, page_copy, paged_append, paged_attention,
                                paged_write, scaled_cos_sin)
from triton_llm.kernels.linear import linear
from triton_llm.pages import PagePool

from .engine import LlamaSession, LlamaWeights


class PagedSession(LlamaSession):
    """Paged KV caches and step buffers for ``batch`` sequences of a model.

    max_seq       longest sequence (positions)
    page_size     tokens of a page
    n_pages       pages of the arena (default: enough for every sequence at
                  max_seq); a step that needs more raises RuntimeError
    window, sinks
                  window > 0: every token sees the last ``window`` tokens, itself
                  among them, and the first ``sinks``
    rope_scaling  see ``scaled_cos_sin``: positions past the model's window

    The other arguments are LlamaSession's. ``step`` (or ``decode_step``)
    advances every slot that holds a sequence; the others run idle, on one page
    past the pool's that they share. Where pages run out, the slots that were to
    get some hold no sequence afterwards; the others are as they were.
    """

    def __init__(self, wts: LlamaWeights, batch: int, max_seq: int, page_size: int = 64,
                 n_pages: int | None = None, window: int = 0, sinks: int = 0,
                 rope_scaling=None, **kw):
        if page_size < 1:
            raise ValueError(f"page_size must be >= 1, got {page_size}")
        if window < 0 or sinks < 0 or (sinks and not window):
            raise ValueError(f"window ({window}) and sinks ({sinks}) must be >= 0, and "
                             "sinks need a window")
        if wts.D % 16:
            raise ValueError(f"head_dim ({wts.D}) must be a multiple of 16")
        self.P, self.window, self.sinks = int(page_size), int(window), int(sinks)
        self.rope_scaling = rope_scaling
        self.cols = -(-int(max_seq) // self.P)
        self.n_pages = int(batch) * self.cols if n_pages is None else int(n_pages)
        super().__init__(wts, batch, max_seq, **kw)

    def _rope_tables(self):
        if self.rope_scaling is None:
            return super()._rope_tables()
        cos, sin = scaled_cos_sin(self.S, self.w.D, self.w.config.rope_theta,
                                  self.rope_scaling)
        return gpu.to_device(cos), gpu.to_device(sin)

    def _cache_buffers(self):
        w = self.w
        shape = (2 * w.L, self.n_pages + 1, w.Hkv, self.P, w.D)   # (the last: idle slots)
        self.arena = gpu.allocate(shape, "bfloat16" if self.kv_bf16 else np.float32)
        self.pool = PagePool(self.n_pages)
        self._table = np.full((self.B, self.cols), -1, np.int32)
        self._table[:, 0] = self.n_pages
        self.table = gpu.to_device(self._table)
        plane = self.arena.nbytes // (2 * w.L)
        self.pages = [PagedKV(gpu.sub_view(self.arena, 2 * i * plane, shape[1:]),
                              gpu.sub_view(self.arena, (2 * i + 1) * plane, shape[1:]),
                              self.table) for i in range(w.L)]
        self.kv = None                            # one layer's staging of a prefill
        self._pos = np.zeros(self.B, np.int64)    # next positions
        self._live = np.zeros(self.B, bool)       # slots that hold a sequence
        self._fixed = False                       # pages reserved, tables on the device
        self._capturing = False
        self.qkv = gpu.allocate((self.B, (w.H + 2 * w.Hkv) * w.D), np.float32)
        self.attn_ws = PagedWorkspace(self.B, w.H, w.Hkv, w.D)
        self._prompt_ws = None                    # of windowed prompts, and its rows
        self._prompt_ws_rows = 0

    def _upload(self):
        self.table.from_numpy(self._table)

    # -- pages ------------------------------------------------------------
    def _drop(self, row, which) -> None:
        """Gives back the pages of these columns of a table row."""
        pages = row[which & (row >= 0)]
        self.pool.release(pages[pages < self.n_pages])
        row[which] = -1

    def _idle(self, slots) -> None:
        """Slots without a sequence: no pages of the pool, position 0."""
        for b in slots:
            self._drop(self._table[b], np.ones(self.cols, bool))
            self._table[b, 0] = self.n_pages
            self._live[b], self._pos[b] = False, 0

    def _set_pages(self, slots, tokens):
        """Fresh pages for new sequences of these lengths."""
        self._idle(slots)
        need = [max(1, -(-int(n) // self.P)) for n in tokens]
        if sum(need) > self.pool.free:
            self._upload_all()
            self.pool.take(sum(need))   # (raises)
        for b, n in zip(slots, need):
            self._table[b, :n] = self.pool.take(n)
            self._live[b] = True
        self._upload()

    def _upload_all(self):
        self._upload()
        # (idle slots' positions are theirs, not the last prefill's)
        for t in (self.pos, self.lens):
            t.from_numpy(self._pos.astype(np.int32))

    def _outside(self, length: int) -> np.ndarray:
        """Columns whose tokens a row of this length does not see."""
        first = np.arange(self.cols) * self.P
        return (first >= self.sinks) & (first + self.P <= length - self.window)

    def _drop_outside(self, slot: int, length: int) -> bool:
        if not self.window:
            return False
        row = self._table[slot]
        old = self._outside(length) & (row >= 0)
        self._drop(row, old)
        return bool(old.any())

    def _advance(self):
        """Pages for the tokens that the next step writes."""
        if self._fixed:
            self._pos += 1
            return
        # (idle slots stay within their page, and where sequences may be)
        idle = ~self._live & (self._pos >= min(self.P, self.S))
        if (self._live & (self._pos >= self.S)).any():
            raise ValueError(f"a sequence has reached max_seq ({self.S})")
        if idle.any():
            self._pos[idle] = 0
            self._upload_all()
        changed = False
        try:
            for b in np.flatnonzero(self._live & (self._pos % self.P == 0)):
                changed |= self._drop_outside(b, int(self._pos[b]) + 1)
                if self._table[b, self._pos[b] // self.P] < 0:
                    self._table[b, self._pos[b] // self.P] = self.pool.take(1)[0]
                    changed = True
        finally:   # (a caller may release a slot and go on where pages ran out)
            if changed:
                self._upload()
        self._keys_hint = int(self._pos[self._live].sum()) + self.B
        self._pos += 1

    def release(self, slots) -> None:
        """Ends the sequences in ``slots`` and frees their pages."""
        slots = [int(b) for b in np.asarray(slots, np.int64).reshape(-1)]
        if not all(0 <= b < self.B for b in slots):
            raise ValueError(f"slots {slots} are not all in the batch of {self.B}")
        self._idle(slots)
        self._upload_all()

    def fork(self, src: int, dst, reserve: int = 0) -> None:
        """Continues the sequence of slot ``src`` in the slots ``dst`` as well:
        full pages are shared, the tokens of the last page are copied.
        ``reserve``: tokens that every one of them, ``src`` too, gets its own
        pages for ahead of time."""
        dst = [int(d) for d in np.asarray(dst, np.int64).reshape(-1)]
        if not all(0 <= b < self.B for b in [src, *dst]) or not self._live[src] or \
                src in dst or len(set(dst)) != len(dst):
            raise ValueError(f"cannot fork slot {src} into {dst}")
        pos = int(self._pos[src])
        full, part = divmod(pos, self.P)
        last = min(self.cols, max(full + (part > 0), -(-(pos + reserve) // self.P)))
        self._idle(dst)
        more = np.flatnonzero(self._table[src, full:last] < 0) + full
        need = len(dst) * (last - full) + len(more)
        if need > self.pool.free:
            self._upload_all()
            self.pool.take(need)   # (raises)
        copies = []
        shared = self._table[src, :full]
        for d in dst:
            self.pool.share(shared[shared >= 0])
            self._table[d, 0] = -1
            self._table[d, :full] = shared
            self._table[d, full:last] = self.pool.take(last - full)
            if part:
                copies.append((self._table[src, full], self._table[d, full], part))
            self._live[d], self._pos[d] = True, pos
        self._table[src, more] = self.pool.take(len(more))
        self._upload_all()
        if copies:
            c = np.array(copies, np.int32).T.copy()
            page_copy(self.arena, *[gpu.to_device(x) for x in c])
        ids = self.ids.to_numpy()
        ids[dst] = ids[src]
        self.ids.from_numpy(ids)

    def compact(self) -> int:
        """Moves the used pages to the front of the arena; returns how many
        moved."""
        src, dst, where = self.pool.compact()
        if len(src):
            page_copy(self.arena, gpu.to_device(src), gpu.to_device(dst))
            where = np.append(where, [self.n_pages, -1])   # the idle slots' page, none
            self._table = where[self._table].astype(np.int32)
            self._upload()
        return len(src)

    # -- one layer ----------------------------------------------------------
    def _prompt_seqs(self, slots, lens, pos):
        # one after another in the staging cache; their rows' slots for the pages
        k, at = self.kv[0][0], np.arange(len(slots), dtype=np.int32)
        self._p_slot = gpu.to_device(np.repeat(slots, lens).astype(np.int32))
        self._p_src = gpu.to_device((np.repeat(at, lens).astype(np.int64) * k.shape[1]
                                     * k.shape[2] + pos).astype(np.int32))
        return at

    def _project_qkv(self, i, M, x, q, row_seq, row_pos, lens, ws, decode, fold_in):
        w = self.w
        if decode:
            linear(x, w.layers[i]["qkv"], out_dev=self.qkv, ws=ws, M=M, fold_in=fold_in)
            paged_append(self.pages[i], self.qkv, row_pos, q, self.cos, self.sin,
                         n_head=w.H, blocked=True, lens_out=lens, rows=M)
            return
        super()._project_qkv(i, M, x, q, row_seq, row_pos, lens, ws, decode, fold_in)
        k, v = self.kv[i]
        paged_write(self.pages[i], k, v, gpu.sub_view(row_pos, 0, (M,)),
                    row_seq=self._p_slot, row_src=self._p_src,
                    row_stride=w.D, head_stride=int(k.shape[2]) * w.D)

    def _attend(self, i, M, q, attn, row_seq, lens, decode, attn_ws, row_len, max_len):
        w = self.w
        if decode:
            paged_attention(self.pages[i], q, lens, attn, max_len=self.S,
                            keys_hint=self._keys_hint, window=self.window,
                            sinks=self.sinks, workspace=attn_ws)
        elif self.window:
            # prompt rows over their windows
            if M > self._prompt_ws_rows:
                self._prompt_ws = PagedWorkspace(M, w.H, w.Hkv, w.D)
                self._prompt_ws_rows = M
            paged_attention(self.pages[i], gpu.sub_view(q, 0, (M, w.H, w.D)),
                            gpu.sub_view(row_len, 0, (M,)), attn,
                            row_seq=self._p_slot, max_len=max_len, window=self.window,
                            sinks=self.sinks, workspace=self._prompt_ws)
        else:
            super()._attend(i, M, q, attn, row_seq, lens, decode, attn_ws, row_len, max_len)

    # -- steps ----------------------------------------------------------------
    def prefill(self, prompts, all_logits=False, slots=None):
        """``LlamaSession.prefill`` into pages; every slot's old sequence ends."""
        prompts, at, lens, keep = self._check_prompts(prompts, slots)
        if self._fixed:
            raise RuntimeError("the session's pages are reserved by a beam search")
        if not keep:
            self._idle(np.setdiff1d(np.arange(self.B), at))
        self._set_pages(at, lens)
        w = self.w
        shape = (len(at), w.Hkv, int(lens.max()), w.D)
        dt = "bfloat16" if self.kv_bf16 else np.float32
        try:
            self.kv = [(gpu.allocate(shape, dt), gpu.allocate(shape, dt))] * w.L
            out = super().prefill(prompts, all_logits, slots)
        except BaseException:
            self.release(at)
            raise
        finally:
            self.kv = self._p_src = self._p_slot = None
        self._pos[at] = lens
        for b, n in zip(at, lens):
            self._drop_outside(int(b), int(n) + 1)
        self._upload_all()
        return out

    def set_state(self, pos, ids):
        """Sequences of these lengths with whatever their pages hold."""
        pos = np.asarray(pos, np.int64)
        if pos.shape != (self.B,) or np.shape(ids) != (self.B,) or (pos < 0).any() or \
                (pos > self.S).any():
            raise ValueError(f"set_state needs {self.B} lengths within max_seq ({self.S}) "
                             f"and as many tokens, got {pos.tolist()}, {np.shape(ids)}")
        self._set_pages(range(len(pos)), pos)
        for b, n in enumerate(pos):
            self._drop_outside(b, int(n) + 1)
        self._pos[:] = pos
        self._upload()
        super().set_state(pos, ids)

    def decode_step(self, sample=True, temperature=0.0, top_k=0):
        if not self._capturing:
            self._advance()
        return super().decode_step(sample, temperature, top_k) + self.w.L

    def capture(self):
        self._capturing = True
        try:
            return super().capture()
        finally:
            self._capturing = False

    def step(self):
        if self.graph is not None:
            self._advance()
            self.graph.launch()
        else:
            self.decode_step(True)


def beam_search(wts: LlamaWeights, prompts, beams: int, max_new_tokens: int,
                eos_token_id: int | None = None, length_penalty: float = 0.0,
                use_graph: bool = True, **session):
    """The ``beams`` best continuations of every prompt.

    Returns for every prompt a list of (generated tokens, score), best first:
    the score is the sum of the tokens' log-probabilities, divided by (number of
    tokens)^length_penalty. A beam ends at ``eos_token_id``. ``session``:
    arguments of PagedSession.
    """
    prompts = [np.asarray(p, np.int32).reshape(-1) for p in prompts]
    G, W = len(prompts), int(beams)
    if not 1 <= W <= 32 or W > wts.V:
        raise ValueError(f"beams must be in [1, 32] and within the vocabulary, got {beams}")
    if max_new_tokens < 1:
        raise ValueError("max_new_tokens must be >= 1")
    if G == 0:
        return []
    longest = max(len(p) for p in prompts) + max_new_tokens
    P = int(session.get("page_size", 64))
    if session.get("window"):
        raise ValueError("beam search keeps every page: no window")
    # a prompt's full pages once, and every beam's own from there on
    own = sum(len(p) // P + W * (-(-(len(p) + max_new_tokens) // P) - len(p) // P)
              for p in prompts)
    session.setdefault("n_pages", own)
    s = PagedSession(wts, G * W, longest, **session)
    first = np.arange(G) * W
    s.prefill(prompts, slots=first)
    # the first step continues the prompts themselves, one beam each
    i32, f32 = np.int32, np.float32
    scores = [gpu.zeros((G, W), f32), gpu.allocate((G, W), f32)]
    parents, tokens = gpu.allocate((G, W), i32), gpu.allocate((G, W), i32)
    done, done_out = gpu.zeros((G, W), i32), gpu.allocate((G, W), i32)
    eos = -1 if eos_token_id is None else int(eos_token_id)
    pad = max(eos, 0)
    beam_select(gpu.sub_view(s.logits, 0, (G, wts.V)), gpu.zeros((G, 1), f32), scores[0],
                parents, tokens, pad_token=pad, out_done=done, eos_token=eos)
    for g in range(G):
        s.fork(int(first[g]), first[g] + np.arange(1, W), reserve=max_new_tokens)
    s._fixed = True
    gpu.copy_d2d(s.ids, tokens)
    found = [[[int(t)] for t in row] for row in tokens.to_numpy()]
    ends = done.to_numpy() != 0

    ws = BeamWorkspace(G, W, wts.V, W)
    copies = [gpu.allocate((G * W,), i32) for _ in range(3)]

    def advance():
        s.decode_step(sample=False)
        beam_select(s.logits, scores[0], scores[1], parents, tokens, done=done,
                    pad_token=pad, out_done=done_out, eos_token=eos, workspace=ws)
        beam_reorder(parents, s.lens, s.table, s.table, *copies, page_size=s.P)
        page_copy(s.arena, *copies)
        for dst, src in ((scores[0], scores[1]), (done, done_out), (s.ids, tokens),
                         (s.pos, s.lens)):
            gpu.copy_d2d(dst, src)

    graph = None
    for step in range(1, max_new_tokens):
        if ends.all():
            break
        if graph is None and use_graph and step < max_new_tokens - 1:
            s._capturing = True
            graph = gpu.Graph()
            with graph:
                advance()
            s._capturing = False
        if graph is not None:
            graph.launch()
        else:
            advance()
        up, tok = parents.to_numpy(), tokens.to_numpy()
        found = [[found[g][up[g, b]] + ([] if ends[g, up[g, b]] else [int(tok[g, b])])
                  for b in range(W)] for g in range(G)]
        ends = done.to_numpy() != 0
    total = scores[0].to_numpy()
    out = []
    for g in range(G):
        ranked = [(np.array(t, np.int32), float(total[g, b]) / len(t) ** length_penalty)
                  for b, t in enumerate(found[g])]
        out.append(sorted(ranked, key=lambda r: -r[1]))
    s.close()
    return out
