"""Operators on a paged KV cache (no counterpart in the reference, whose cache
is one preallocated block per sequence, smollm2_triton/model.py:219-225).

* ``PagedKV``         one layer's K and V pages with the sequences' page tables;
* ``paged_attention`` attention of one new token per row, optionally with a
  sliding window and a few first tokens that stay visible;
* ``paged_append``    rotary positions on new rows' q and k, and k / v written
  into their pages; ``paged_write`` the same for separate k and v;
* ``page_copy``       page copies over every plane of an arena.

Tensors are ``DeviceTensor``s, or any object with ``data_ptr()``, ``shape`` and
``dtype`` on the same GPU. Calls run on the library stream unless ``stream``
(a CUDA stream handle) is given; work of another stream on the same tensors has
to be ordered by the caller.
"""

from __future__ import annotations

import ctypes
import math

from triton_llm import gpu, _lib
from ._common import dtype_code, on_device, require_gpu, strides


class PagedKV:
    """K and V pages of one layer and the page tables of its sequences.

    k_pages, v_pages
        fp32 or bf16, (n_pages, n_kv_head, page_size, head_dim), or with
        ``slots_first`` (n_pages, page_size, n_kv_head, head_dim). Only the last
        axis has to be contiguous.
    table
        (n_seq, pages) int32 on the device: token j of sequence s is slot
        j % page_size of page ``table[s, j // page_size]``. Entries that no call
        needs may hold anything.

    The object keeps its tensors alive; it is built once and used for every
    call on the layer.
    """

    def __init__(self, k_pages, v_pages, table, slots_first=False):
        if len(k_pages.shape) != 4 or tuple(v_pages.shape) != tuple(k_pages.shape):
            raise ValueError(f"k_pages and v_pages must be 4D with the same shape, got "
                             f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
        code = dtype_code(k_pages, "k_pages")
        if code not in (_lib.F32, _lib.BF16) or dtype_code(v_pages, "v_pages") != code:
            raise ValueError(f"k_pages and v_pages must both be float32 or bfloat16, got "
                             f"{k_pages.dtype} and {v_pages.dtype}")
        sk, sv = strides(k_pages), strides(v_pages)
        if sk != sv:
            raise ValueError(f"k_pages and v_pages have different strides: {sk}, {sv}")
        if sk[3] != 1 and k_pages.shape[3] > 1:
            raise ValueError("the last axis of k_pages and v_pages must be contiguous")
        if len(table.shape) != 2:
            raise ValueError(f"table must be 2D, got {tuple(table.shape)}")
        if dtype_code(table, "table") != _lib.I32:
            raise ValueError(f"table must be int32, got {table.dtype}")
        for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages"), (table, "table")):
            require_gpu(t, name)
        st = strides(table)
        if st[1] != 1 and table.shape[1] > 1:
            raise ValueError("rows of the page table must be contiguous")
        self.k, self.v, self.table = k_pages, v_pages, table
        self.slots_first = bool(slots_first)
        a, b = (2, 1) if slots_first else (1, 2)
        self.n_pages = int(k_pages.shape[0])
        self.n_kv_head, self.page_size = int(k_pages.shape[a]), int(k_pages.shape[b])
        self.head_dim = int(k_pages.shape[3])
        self.n_seq, self.columns = int(table.shape[0]), int(table.shape[1])
        self.dtype = code
        self.device = None   # of the library stream's workspaces, once needed
        self._c = _lib.PagedKVStruct(
            k_pages.data_ptr(), v_pages.data_ptr(), code, self.n_pages, self.page_size,
            self.n_kv_head, self.head_dim, self.n_seq, self.columns, 0, sk[0], sk[a],
            sk[b], st[0], table.data_ptr())
        self._ref = ctypes.addressof(self._c)


class PagedWorkspace:
    """Scratch of ``paged_attention`` for up to ``rows`` rows (allocated once;
    calls that overlap on the GPU need one each). Ready for any stream when it has
    been made, and released only after the device's work."""

    def __init__(self, rows, n_head, n_kv_head, head_dim):
        pb, cb = ctypes.c_size_t(), ctypes.c_size_t()
        _lib.call("tllm_paged_attention_workspace", int(rows), int(n_head),
                  int(n_kv_head), int(head_dim), ctypes.byref(pb), ctypes.byref(cb))
        self.key = (int(rows), int(n_head), int(n_kv_head), int(head_dim))
        at = -(-cb.value // 256) * 256   # counters, then the partials
        self._buf = gpu.Scratch(at + pb.value, zeros=at)
        self.counters, self.counter_bytes = self._buf.data_ptr(), cb.value
        self.partial, self.partial_bytes = self.counters + at, pb.value


_workspaces: dict = {}


def _workspace(make, *key):
    """The library stream's own workspace of a device: calls on that stream run
    one after another, so they can share it."""
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = make()
    return ws


def _out_args(out, rows, n_head, head_dim):
    """(address, dtype code, plane rows, row stride, head stride) of an
    attention output: fp32 or bf16 (rows, n_head, head_dim), or a buffer of at
    least so many rows and n_head * head_dim columns: fp32 2D, or in an operand
    format (``gpu.act_empty``)."""
    code = dtype_code(out, "out")
    if code == _lib.I32:
        raise ValueError("out must be float32 or bfloat16")
    if type(out) is gpu.DeviceTensor and (out.is_split or len(out.shape) == 2):
        prows, cols = out.shape[-2:]
        if prows < rows or cols < n_head * head_dim:
            raise ValueError(f"out holds {prows} rows of {cols}, {rows} of "
                             f"{n_head * head_dim} needed")
        if out.is_split and out.shape[0] == 2:
            code = _lib.SPLIT
        return out.data_ptr(), code, prows, cols, head_dim
    ptr = on_device(out, "out", None, (rows, n_head, head_dim))
    return ptr, code, rows, n_head * head_dim, head_dim


def paged_attention(kv, q, row_len, out, row_seq=None, max_len=0, keys_hint=0, window=0,
                    sinks=0, sm_scale=None, workspace=None, stream=None):
    """Attention of one token per row over a paged cache.

    kv        PagedKV
    q         (rows, n_head, head_dim) float32, the last axis contiguous
    row_len   (rows,) int32 on the device: keys before and with the row's token
    out       (rows, n_head, head_dim) float32 or bfloat16, or a buffer of at least
              rows x (n_head * head_dim): fp32, or in an operand format
    row_seq   (rows,) int32 on the device: the rows' sequences (None: row r is
              sequence r); rows may share a sequence
    max_len, keys_hint
              the longest row and the sum of the lengths, as far as the host
              knows them: they plan how the work is split, never the result
    window, sinks
              window > 0: a row sees its last ``window`` keys and the first
              ``sinks`` ones; pages outside them are not read
    workspace PagedWorkspace, needed with ``stream``; without one the library
              stream's own is used (made by the first call of a shape: before a
              graph capture, not in it)

    A row without a visible key gives zeros. Returns ``out``.
    """
    shape = q.shape
    if len(shape) != 3 or shape[2] != kv.head_dim:
        raise ValueError(f"q must be (rows, n_head, {kv.head_dim}), got {tuple(shape)}")
    rows, n_head, _ = shape
    if dtype_code(q, "q") != _lib.F32:
        raise ValueError(f"q must be float32, got {q.dtype}")
    sq = strides(q)
    if sq[2] != 1 and kv.head_dim > 1:
        raise ValueError("the last axis of q must be contiguous")
    require_gpu(q, "q")
    o = _out_args(out, rows, n_head, kv.head_dim)
    if n_head % kv.n_kv_head:
        raise ValueError(f"n_head ({n_head}) must be divisible by n_kv_head ({kv.n_kv_head})")
    lens = on_device(row_len, "row_len", _lib.I32, (rows,))
    seq = 0 if row_seq is None else on_device(row_seq, "row_seq", _lib.I32, (rows,))
    if workspace is None:
        if stream is not None:
            raise ValueError("a call on another stream needs its own workspace")
        if kv.device is None:
            kv.device = gpu.current_device()
        n = 1 << max(0, rows - 1).bit_length()
        workspace = _workspace(
            lambda: PagedWorkspace(n, n_head, kv.n_kv_head, kv.head_dim),
            "attention", kv.device, n, n_head, kv.n_kv_head, kv.head_dim)
    _lib.call("tllm_paged_attention", kv._ref, _lib.PAGED_ATTN.pack(
        q.data_ptr(), seq, lens, o[0], workspace.partial, workspace.counters,
        workspace.partial_bytes, workspace.counter_bytes, sq[0], sq[1], o[2], o[3], o[4],
        int(keys_hint), o[1], rows, n_head, int(max_len), int(window), int(sinks),
        float(sm_scale or 0.0), 0), stream)
    return out


def _tables(cos, sin):
    """(cos, sin, positions, rotary values) of rotary tables, zeros for none."""
    if cos is None and sin is None:
        return 0, 0, 0, 0
    if cos is None or sin is None:
        raise ValueError("cos and sin go together")
    shape = cos.shape
    if len(shape) != 2 or sin.shape != shape:
        raise ValueError(f"cos and sin must be 2D with the same shape, got "
                         f"{tuple(shape)} and {tuple(sin.shape)}")
    n_pos, half = shape
    return on_device(cos, "cos", _lib.F32), on_device(sin, "sin", _lib.F32), n_pos, 2 * half


def _index(t, name, n):
    return 0 if t is None else on_device(t, name, _lib.I32, (n,))


def paged_append(kv, qkv, row_pos, q_out, cos=None, sin=None, *, n_head, row_seq=None,
                 interleaved=False, blocked=False, lens_out=None, rows=None, stream=None):
    """New tokens of a paged cache from fused projections, with rotary positions.

    qkv      (rows, (n_head + 2 n_kv_head) * head_dim) float32: every row's q,
             k and v heads; with ``blocked`` each head as blocks of 8 values
             (8b.., head_dim/2 + 8b..), the order of ``Linear`` built by
             ``qkv_rows``
    row_pos  (rows,) int32 on the device: positions; row_seq their sequences
             (None: row r is sequence r)
    q_out    (rows, n_head, head_dim) float32: the rotated q
    cos, sin (positions, rotary_dim / 2) float32 tables, or None for no rotation;
             the first rotary_dim values of a head turn, as pairs
             (i, i + rotary_dim / 2) or, ``interleaved``, (2 i, 2 i + 1)
    lens_out (n_seq,) int32 or None: raised to position + 1 at every row's sequence
    rows     use only the first ``rows`` rows
    """
    D, K = kv.head_dim, kv.n_kv_head
    shape, cols = qkv.shape, (n_head + 2 * K) * D
    if len(shape) != 2 or shape[1] != cols:
        raise ValueError(f"qkv must be (rows, {cols}), got {tuple(shape)}")
    src_rows = shape[0]
    if dtype_code(qkv, "qkv") != _lib.F32:
        raise ValueError(f"qkv must be float32, got {qkv.dtype}")
    ld, one = strides(qkv)
    if one != 1:
        raise ValueError("rows of qkv must be contiguous")
    require_gpu(qkv, "qkv")
    n = src_rows if rows is None else int(rows)
    if n > src_rows:
        raise ValueError(f"{n} rows of a qkv of {src_rows}")
    shape = q_out.shape
    if len(shape) != 3 or shape[0] < n or shape[1] != n_head or shape[2] != D:
        raise ValueError(f"q_out must be ({n}, {n_head}, {D}), got {tuple(shape)}")
    cos_t, sin_t, n_pos, rotary = _tables(cos, sin)
    at = qkv.data_ptr()
    r = _lib.PAGED_ROWS.pack(
        at, at + n_head * D * 4, at + (n_head + K) * D * 4,
        on_device(q_out, "q_out", _lib.F32), 0,
        0 if row_seq is None else on_device(row_seq, "row_seq", _lib.I32, (n,)),
        on_device(row_pos, "row_pos", _lib.I32, (n,)),
        0 if lens_out is None else on_device(lens_out, "lens_out", _lib.I32, (kv.n_seq,)),
        cos_t, sin_t, ld, D, ld, D, ld, D, n_head * D, D, _lib.F32, n, n_head, rotary,
        n_pos, bool(interleaved), bool(blocked), src_rows)
    _lib.call("tllm_paged_append", kv._ref, r, stream)
    return q_out


def paged_write(kv, k, v, row_pos, row_seq=None, row_src=None, cos=None, sin=None,
                interleaved=False, lens_out=None, row_stride=None, head_stride=None,
                stream=None):
    """k and v rows into the pages of a paged cache.

    k, v     fp32 or bf16, (rows, n_kv_head, head_dim), the last axis contiguous;
             with row_stride and head_stride (elements) any buffers in which
             row i, head h starts at i * row_stride + h * head_stride
    row_src  (rows,) int32 on the device: the source row of every row written
             (None: the rows in order)
    The other arguments as for ``paged_append``.
    """
    code = dtype_code(k, "k")
    if code not in (_lib.F32, _lib.BF16) or dtype_code(v, "v") != code:
        raise ValueError(f"k and v must both be float32 or bfloat16, got {k.dtype}, {v.dtype}")
    if len(row_pos.shape) != 1:
        raise ValueError(f"row_pos must be 1D, got {tuple(row_pos.shape)}")
    n = int(row_pos.shape[0])
    if (row_stride is None) != (head_stride is None):
        raise ValueError("row_stride and head_stride go together")
    if row_stride is None:
        for t, name in ((k, "k"), (v, "v")):
            if len(t.shape) != 3 or tuple(t.shape[1:]) != (kv.n_kv_head, kv.head_dim):
                raise ValueError(f"{name} must be (rows, {kv.n_kv_head}, {kv.head_dim}), "
                                 f"got {tuple(t.shape)}")
            if row_src is None and t.shape[0] != n:
                raise ValueError(f"{name} has {t.shape[0]} rows, row_pos {n}")
        sk, sv = strides(k), strides(v)
        if sk[2] != 1 or sv[2] != 1:
            raise ValueError("the last axis of k and v must be contiguous")
        src_rows = min(int(k.shape[0]), int(v.shape[0]))
    else:
        sk = sv = (int(row_stride), int(head_stride))
        if sk[0] < 1 or sk[1] < 0:
            raise ValueError(f"row_stride ({sk[0]}) must be >= 1, head_stride ({sk[1]}) >= 0")
        for t, name in ((k, "k"), (v, "v")):
            on_device(t, name)
        values = min(math.prod(k.shape), math.prod(v.shape))
        src_rows = max(0, values - (kv.n_kv_head - 1) * sk[1] - kv.head_dim + sk[0]) // sk[0]
        if n and src_rows == 0:
            raise ValueError("k and v hold no row of these strides")
    require_gpu(k, "k")
    require_gpu(v, "v")
    cos_t, sin_t, n_pos, rotary = _tables(cos, sin)
    r = _lib.PAGED_ROWS.pack(
        0, k.data_ptr(), v.data_ptr(), 0, _index(row_src, "row_src", n),
        _index(row_seq, "row_seq", n), _index(row_pos, "row_pos", n),
        _index(lens_out, "lens_out", kv.n_seq),
        cos_t, sin_t, 0, 0, sk[0], sk[1], sv[0], sv[1], 0, 0, code, n, 0, rotary, n_pos,
        bool(interleaved), 0, src_rows)
    _lib.call("tllm_paged_append", kv._ref, r, stream)


def page_copy(arena, src, dst, fill=None, slots_first=False, stream=None):
    """Copies pages over every plane of an arena: for each i the first
    ``fill[i]`` slots (None: all) of page ``src[i]`` to page ``dst[i]``.

    arena  (planes, n_pages, n_kv_head, page_size, head_dim), or with
           ``slots_first`` (planes, n_pages, page_size, n_kv_head, head_dim);
           fp32 or bf16, contiguous (K and V of every layer are its planes)
    src, dst, fill
           (copies,) int32 on the device; a copy with src == dst or a negative
           page does nothing. No page may be written twice, or written and read.
    """
    if len(arena.shape) != 5:
        raise ValueError(f"arena must be 5D, got {tuple(arena.shape)}")
    planes, pages, a, b, D = (int(x) for x in arena.shape)
    code = dtype_code(arena, "arena")
    if code == _lib.I32:
        raise ValueError("arena must be float32 or bfloat16")
    size = 2 if code == _lib.BF16 else 4
    base = on_device(arena, "arena")
    if len(src.shape) != 1:
        raise ValueError(f"src must be 1D, got {tuple(src.shape)}")
    n = int(src.shape[0])
    f = None if fill is None else on_device(fill, "fill", _lib.I32, (n,))
    page = a * b * D * size
    heads, run, slots, row = (1, 0, a, b * D * size) if slots_first else \
        (a, b * D * size, b, D * size)
    _lib.call("tllm_page_copy", base, pages * page, planes, page, pages, heads, run, slots,
              row, on_device(src, "src", _lib.I32), on_device(dst, "dst", _lib.I32, (n,)),
              f, n, stream)
