"""Refusals of the paged-cache operators: everything here is refused on the
host, before any device work (CPU-only)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from triton_llm import _lib
from triton_llm.kernels import (PagedKV, beam_reorder, beam_select, page_copy, paged_append,
                                paged_attention, paged_write)


class Fake:
    """A tensor that is only described: no call here may reach the device."""

    def __init__(self, shape, dtype="float32", ptr=4096, stride=None, cuda=True):
        self.shape, self.ptr, self.is_cuda = tuple(shape), ptr, cuda
        self.dtype = np.dtype(np.float64) if dtype == "float64" else f"any.{dtype}"
        n = 1
        rev = []
        for s in reversed(self.shape):
            rev.append(n)
            n *= s
        self._stride = stride or tuple(reversed(rev))
        self._packed = stride is None

    def data_ptr(self):
        return self.ptr

    def stride(self):
        return self._stride

    def is_contiguous(self):
        return self._packed


class Scratch:
    partial = counters = 0
    partial_bytes = counter_bytes = 0


class NoCounters:
    partial = counters = 4096
    partial_bytes, counter_bytes = 1 << 30, 0


def kv(n=8, K=2, P=16, D=64, dtype="bfloat16", S=3, C=4, **kw):
    return PagedKV(Fake((n, K, P, D), dtype), Fake((n, K, P, D), dtype),
                   Fake((S, C), "int32"), **kw)


@pytest.mark.parametrize("make,msg", [
    (lambda: PagedKV(Fake((2, 3, 4)), Fake((2, 3, 4)), Fake((1, 1), "int32")), "4D"),
    (lambda: PagedKV(Fake((2, 3, 4, 8)), Fake((2, 3, 4, 16)), Fake((1, 1), "int32")), "same shape"),
    (lambda: PagedKV(Fake((2, 3, 4, 8)), Fake((2, 3, 4, 8), "bfloat16"),
                     Fake((1, 1), "int32")), "both be"),
    (lambda: PagedKV(Fake((2, 3, 4, 8), "float64"), Fake((2, 3, 4, 8), "float64"),
                     Fake((1, 1), "int32")), "float32, bfloat16"),
    (lambda: PagedKV(Fake((2, 3, 4, 8)), Fake((2, 3, 4, 8), stride=(192, 64, 16, 1)),
                     Fake((1, 1), "int32")), "different strides"),
    (lambda: PagedKV(*[Fake((2, 3, 4, 8), stride=(96, 32, 1, 4))] * 2,
                     Fake((1, 1), "int32")), "last axis"),
    (lambda: PagedKV(*[Fake((2, 3, 4, 8))] * 2, Fake((1,), "int32")), "2D"),
    (lambda: PagedKV(*[Fake((2, 3, 4, 8))] * 2, Fake((1, 1))), "int32"),
    (lambda: PagedKV(*[Fake((2, 3, 4, 8), cuda=False)] * 2, Fake((1, 1), "int32")), "GPU"),
])
def test_cache_refusals(make, msg):
    with pytest.raises(ValueError, match=msg):
        make()


def attend(q=(3, 4, 64), lens=(3,), out=(3, 4, 64), cache=None, q_dtype="float32",
           out_dtype="float32", q_ptr=4096, q_stride=None, **kw):
    return paged_attention(cache or kv(), Fake(q, q_dtype, q_ptr, q_stride),
                           Fake(lens, "int32"), Fake(out, out_dtype),
                           **{"workspace": Scratch, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(q=(3, 4, 32)), "q must be"),
    (dict(q_dtype="bfloat16"), "q must be float32"),
    (dict(q=(3, 5, 64), out=(3, 5, 64)), "divisible"),
    (dict(lens=(2,)), "row_len has shape"),
    (dict(out=(3, 4, 32)), "out has shape"),
    (dict(out_dtype="int32"), "out must be"),
    (dict(row_seq=Fake((2,), "int32")), "row_seq has shape"),
    (dict(row_seq=Fake((3,))), "row_seq has dtype"),
    (dict(q=(4, 4, 64), lens=(4,), out=(4, 4, 64)), "4 rows for a table of 3"),
    (dict(window=-1), "window"),
    (dict(sinks=4), "need a window"),
    (dict(max_len=-1), "max_len"),
    (dict(q_ptr=4100), "16-byte aligned"),
    (dict(q_stride=(256, 64, 2)), "last axis"),
    (dict(q_stride=(258, 64, 1)), "whole 16 bytes"),
    (dict(cache=kv(D=60), q=(3, 4, 60), out=(3, 4, 60)), "16-byte units"),
    (dict(cache=kv(D=520), q=(3, 4, 520), out=(3, 4, 520)), "at most 512"),
    (dict(cache=kv(P=1 << 29)), "2.30"),
    (dict(cache=kv(P=4096, C=64), workspace=NoCounters), "counters hold 0 bytes"),
])
def test_attention_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        attend(**kw)


def test_attention_on_another_stream_needs_a_workspace():
    with pytest.raises(ValueError, match="workspace"):
        paged_attention(kv(), Fake((3, 4, 64)), Fake((3,), "int32"), Fake((3, 4, 64)),
                        stream=4096)


def test_attention_of_no_rows():
    attend(q=(0, 4, 64), lens=(0,), out=(0, 4, 64))


def test_workspace_shapes():
    lib = _lib.load()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    ref = ctypes.byref
    assert lib.tllm_paged_attention_workspace(4, 9, 2, 64, ref(a), ref(b)) == _lib.ERR_INVALID_ARG
    assert lib.tllm_paged_attention_workspace(4, 9, 3, 64, ref(a), ref(b)) == _lib.OK
    assert a.value > 0 and b.value >= 4 * 9 * 4
    for args in [(1, 33, 100, 4), (1, 0, 100, 4), (1, 4, 100, 65), (1, 4, 3, 4), (1, 4, 100, 0),
                 (-1, 4, 100, 4), (1, 4, 1 << 27, 4)]:
        assert lib.tllm_beam_workspace(*args, ref(a)) == _lib.ERR_INVALID_ARG


def append(qkv=(3, 8 * 64), pos=(3,), q_out=(3, 4, 64), cos=(10, 32), sin=(10, 32),
           cache=None, n_head=4, qkv_dtype="float32", **kw):
    return paged_append(cache or kv(), Fake(qkv, qkv_dtype), Fake(pos, "int32"), Fake(q_out),
                        cos and Fake(cos), sin and Fake(sin), n_head=n_head, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(qkv=(3, 7 * 64)), "qkv must be"),
    (dict(qkv_dtype="bfloat16"), "qkv must be float32"),
    (dict(pos=(4,)), "row_pos has shape"),
    (dict(q_out=(3, 4, 32)), "q_out must be"),
    (dict(sin=None), "go together"),
    (dict(sin=(10, 16)), "same shape"),
    (dict(cos=(10, 33), sin=(10, 33)), "rotary_dim"),
    (dict(cos=(0, 32), sin=(0, 32)), "n_pos"),
    (dict(rows=4), "4 rows of a qkv of 3"),
    (dict(lens_out=Fake((2,), "int32")), "lens_out has shape"),
    (dict(qkv=(4, 8 * 64), pos=(4,), q_out=(4, 4, 64)), "4 rows for a table of 3"),
    (dict(cache=kv(D=72), qkv=(3, 8 * 72), q_out=(3, 4, 72), cos=None, sin=None,
          blocked=True), "blocked"),
])
def test_append_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        append(**kw)


@pytest.mark.parametrize("k,v,pos,kw,msg", [
    ((3, 2, 32), (3, 2, 64), (3,), {}, "k must be"),
    ((3, 2, 64), (2, 2, 64), (3,), {}, "v has 2 rows"),
    ((3, 2, 64), (3, 2, 64), (3,), dict(row_stride=64), "go together"),
    ((3, 2, 64), (3, 2, 64), (3, 1), {}, "1D"),
    ((3, 2, 64), (3, 2, 64), (4,), dict(row_stride=128, head_stride=64), "4 rows of 3 source"),
    ((1, 1, 64), (3, 2, 64), (3,), dict(row_stride=128, head_stride=64), "no row"),
    ((3, 2, 64), (3, 2, 64), (3,), dict(row_stride=0, head_stride=64), "row_stride"),
])
def test_write_refusals(k, v, pos, kw, msg):
    with pytest.raises(ValueError, match=msg):
        paged_write(kv(), Fake(k), Fake(v), Fake(pos, "int32"), **kw)


def test_append_in_place_refusals():
    c, r = kv(), _lib.PagedRowsStruct()
    r.q = r.q_out = r.k = r.v = r.row_pos = 4096
    r.rows, r.n_head, r.q_row_stride, r.q_out_row_stride = 1, 4, 512, 256
    assert _lib.load().tllm_paged_append(c._ref, ctypes.addressof(r), None) == _lib.ERR_INVALID_ARG
    assert "in place" in _lib.last_error()


@pytest.mark.parametrize("arena,src,dst,fill,dtype,msg", [
    ((2, 3, 4, 5), (1,), (1,), None, "float32", "5D"),
    ((2, 3, 4, 5, 6), (1, 1), (1,), None, "float32", "1D"),
    ((2, 3, 4, 5, 6), (2,), (1,), None, "float32", "dst has shape"),
    ((2, 3, 4, 5, 6), (2,), (2,), (1,), "float32", "fill has shape"),
    ((2, 3, 4, 5, 6), (2,), (2,), None, "int32", "arena must be"),
    ((70000, 3, 4, 5, 6), (2,), (2,), None, "float32", "planes"),
])
def test_copy_refusals(arena, src, dst, fill, dtype, msg):
    with pytest.raises(ValueError, match=msg):
        page_copy(Fake(arena, dtype), Fake(src, "int32"), Fake(dst, "int32"),
                  fill and Fake(fill, "int32"))


def beams(logits=(8, 100), scores=(2, 4), out=(2, 4), tokens=(2, 4), dtype="float32", **kw):
    class Ws:
        ptr, nbytes = 4096, 0
    return beam_select(Fake(logits, dtype), Fake(scores), Fake(out), Fake(out, "int32"),
                       Fake(tokens, "int32"), workspace=Ws, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=(7, 100)), "7 rows"),
    (dict(scores=(8,)), "2D"),
    (dict(dtype="bfloat16"), "logits must be float32"),
    (dict(out=(3, 4)), "out_scores must be"),
    (dict(tokens=(2, 5)), "out_tokens has shape"),
    (dict(out=(2, 65), tokens=(2, 65)), "k "),
    (dict(logits=(8, 3)), "k "),
    (dict(logits=(66, 100), scores=(2, 33)), "beams"),
    (dict(done=Fake((7,), "int32")), "done has 7"),
    (dict(done=Fake((2, 4), "int32"), pad_token=100), "pad_token"),
    (dict(), "workspace of 0 bytes"),
])
def test_beam_select_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        beams(**kw)


@pytest.mark.parametrize("parents,lens,table,out,kw,msg", [
    ((8,), (8,), (8, 3), (8, 3), {}, "2D"),
    ((2, 4), (8,), (7, 3), (7, 3), {}, "7 rows"),
    ((2, 4), (2,), (8, 3), (8, 3), {}, "lens has shape"),
    ((2, 4), (8,), (8, 3), (8, 4), {}, "table_out has shape"),
    ((2, 33), (66,), (66, 3), (66, 3), {}, "beams"),
    ((2, 4), (8,), (8, 3), (8, 3), dict(page_size=0), "0 slots"),
])
def test_beam_reorder_refusals(parents, lens, table, out, kw, msg):
    n = (int(table[0]),)
    c = [Fake(n if len(parents) < 2 else (parents[0] * parents[1],), "int32")
         for _ in range(3)]
    with pytest.raises(ValueError, match=msg):
        beam_reorder(Fake(parents, "int32"), Fake(lens, "int32"), Fake(table, "int32"),
                     Fake(out, "int32"), *c, **dict(dict(page_size=16), **kw))
