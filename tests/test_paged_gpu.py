"""The paged-cache operators on a B200 against plain 64-bit formulas.

Tolerances. q.k is a sum of D <= 512 fp32 products (relative rounding of a sum
of n terms ~ sqrt(n) 2^-24 <= 1.4e-6 of its largest partial sums), the base-2
exponential is good to 2^-22, and the weighted sum of V adds sqrt(keys) 2^-24:
together below 4e-6 of a head's output in the 2-norm. bf16 results may be off
by one rounding, 2^-8 of each value; operand planes (hi + lo) by 2^-16. A
rotated value is two products and a sum: 3 * 2^-24 of the pair's norm. Moved
and unrotated values are exact.
"""

from __future__ import annotations

import numpy as np
import pytest

from triton_llm import gpu
from triton_llm.kernels import (PagedKV, PagedWorkspace, beam_reorder, beam_select,
                                page_copy, paged_append, paged_attention, paged_write)

pytestmark = pytest.mark.gpu

F32_TOL = 4e-6


# -- helpers ----------------------------------------------------------------
def bf16(a):
    return gpu.bf16_bits_to_f32(gpu.f32_to_bf16_bits(a))


def up(a, dtype):
    return gpu.to_device_bf16(a) if dtype == "bf16" else gpu.to_device(a)


def i32(a):
    return gpu.to_device(np.asarray(a, np.int32))


class Cache:
    """Random pages (host copy, NaN where no token lies) and their tables."""

    def __init__(self, lens, K, D, P, dtype, seed=0, slots_first=False, spare=3,
                 window=0, sinks=0):
        rng = np.random.default_rng(seed)
        self.lens, self.P = list(lens), P
        cols = max(1, max(-(-n // P) for n in lens))
        need = [-(-n // P) for n in lens]
        n = sum(need) + spare
        order = rng.permutation(n)
        self.table = np.full((len(lens), cols), -1, np.int32)
        k = np.full((n, K, P, D), np.nan, np.float32)
        v = np.full((n, K, P, D), np.nan, np.float32)
        at = 0
        for s, length in enumerate(lens):
            for c in range(need[s]):
                visible = [j for j in range(c * P, min(length, (c + 1) * P))
                           if not window or j < sinks or j >= length - window]
                if not visible:
                    continue          # a freed page: its entry stays -1
                page = order[at]
                at += 1
                self.table[s, c] = page
                for j in visible:
                    k[page, :, j - c * P] = rng.standard_normal((K, D))
                    v[page, :, j - c * P] = rng.standard_normal((K, D))
        if dtype == "bf16":
            k, v = bf16(k), bf16(v)
        self.k, self.v = k, v
        put = (lambda a: np.ascontiguousarray(a.transpose(0, 2, 1, 3))) if slots_first \
            else (lambda a: a)
        self.kv = PagedKV(up(put(k), dtype), up(put(v), dtype), i32(self.table),
                          slots_first=slots_first)

    def keys(self, seq, at):
        page = self.table[seq, np.asarray(at) // self.P]
        slot = np.asarray(at) % self.P
        return (self.k[page, :, slot].astype(np.float64),
                self.v[page, :, slot].astype(np.float64))


def attend(cache, q, seqs, lens, window=0, sinks=0, scale=None):
    R, H, D = q.shape
    K = cache.k.shape[1]
    scale = scale or D ** -0.5
    out = np.zeros((R, H, D))
    for r in range(R):
        n = lens[r]
        at = [j for j in range(n) if not window or j < sinks or j >= n - window]
        if not at:
            continue
        k, v = cache.keys(seqs[r], at)
        for h in range(H):
            j = h // (H // K)
            s = k[:, j] @ q[r, h].astype(np.float64) * scale
            w = np.exp(s - s.max())
            out[r, h] = w @ v[:, j] / w.sum()
    return out


def head_error(got, want):
    """Largest relative 2-norm error over (row, head); rows of zeros exactly."""
    d = np.linalg.norm(got - want, axis=-1)
    n = np.linalg.norm(want, axis=-1)
    assert np.isfinite(got).all()
    assert (d[n == 0] == 0).all()
    return (d[n > 0] / n[n > 0]).max() if (n > 0).any() else 0.0


def check_attention(H, K, D, P, dtype, lens, window=0, sinks=0, out="f32", seed=0,
                    slots_first=False, **kw):
    cache = Cache(lens, K, D, P, dtype, seed, slots_first, window=window, sinks=sinks)
    rng = np.random.default_rng(seed + 1)
    q = rng.standard_normal((len(lens), H, D)).astype(np.float32)
    want = attend(cache, q, range(len(lens)), lens, window, sinks)
    if out == "f32":
        o, tol = gpu.allocate(q.shape, np.float32), F32_TOL
    elif out == "bf16":
        o, tol = gpu.allocate(q.shape, "bfloat16"), 2.0 ** -8
    else:
        o, tol = gpu.act_empty(len(lens) + 1, H * D, 2), F32_TOL + 2.0 ** -16
    gpu.device_error(reset=True)
    paged_attention(cache.kv, gpu.to_device(q), i32(lens), o, window=window, sinks=sinks,
                    **kw)
    gpu.synchronize()
    if out == "split":
        got = gpu.split_to_host(o, len(lens)).reshape(q.shape)
    else:
        got = gpu.to_host(o)
    assert gpu.device_error() == 0
    err = head_error(got.astype(np.float64), want)
    assert err < tol, f"relative error {err}"


# -- attention --------------------------------------------------------------
LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 1025, 700]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("P", [1, 5, 8, 16, 24, 32, 64, 128, 256])
@pytest.mark.parametrize("H,K,D", [(9, 3, 64), (24, 8, 128)])
def test_attention_page_sizes(H, K, D, P, dtype):
    check_attention(H, K, D, P, dtype, LENS, seed=P)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,K,D", [(1, 1, 8), (5, 5, 16), (2, 1, 32), (12, 12, 64),
                                   (15, 5, 64), (16, 1, 64), (17, 1, 64), (40, 2, 128),
                                   (8, 1, 128), (32, 2, 128), (6, 2, 96), (4, 2, 80),
                                   (3, 1, 256), (2, 2, 512)])
def test_attention_head_layouts(H, K, D, dtype):
    check_attention(H, K, D, 16, dtype, [1, 17, 130, 400], seed=H)


@pytest.mark.parametrize("out", ["f32", "bf16", "split"])
@pytest.mark.parametrize("slots_first", [False, True])
@pytest.mark.parametrize("D,P", [(64, 16), (64, 128), (128, 64), (128, 8), (96, 16)])
def test_attention_layouts_and_outputs(D, P, slots_first, out):
    check_attention(12, 4, D, P, "bf16", [0, 5, 64, 333, 1500], out=out,
                    slots_first=slots_first)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (3, 4), (64, 4), (100, 0),
                                          (130, 70), (1000, 4), (5000, 33)])
@pytest.mark.parametrize("H,K,D,P,dtype", [(9, 3, 64, 16, "bf16"), (24, 8, 128, 64, "bf16"),
                                           (15, 5, 64, 256, "bf16"), (8, 1, 128, 8, "bf16"),
                                           (6, 2, 64, 20, "bf16"), (4, 4, 64, 32, "f32")])
def test_attention_window_and_sinks(H, K, D, P, dtype, window, sinks):
    check_attention(H, K, D, P, dtype, [0, 1, 4, 5, 64, 131, 200, 1100, 2049], window,
                    sinks, seed=window)


@pytest.mark.parametrize("H,K,D,P,dtype", [(24, 8, 128, 64, "bf16"), (9, 3, 64, 16, "bf16"),
                                           (4, 4, 64, 24, "f32")])
@pytest.mark.parametrize("hints", [{}, dict(max_len=20011, keys_hint=20312),
                                   dict(max_len=64), dict(max_len=1, keys_hint=1)])
def test_attention_long_rows_split_and_joined(H, K, D, P, dtype, hints):
    """Many splits, with right, missing and far too small hints."""
    check_attention(H, K, D, P, dtype, [20011, 1, 300], seed=3, **hints)


def test_attention_small_workspace():
    """Scratch for fewer splits than planned gives the same result."""
    ws = PagedWorkspace(3, 9, 3, 64)
    for nbytes in (ws.partial_bytes, 3 * 9 * 2 * 3 * 66 * 4, 0):
        ws.partial_bytes = nbytes
        check_attention(9, 3, 64, 16, "bf16", [5000, 17, 900], workspace=ws)


def test_attention_rows_of_shared_sequences():
    """Rows that name their sequence: prompt rows, shared prefixes."""
    lens = [130, 40]
    cache = Cache(lens, 3, 64, 16, "bf16", 5)
    seqs = [0] * 130 + [1, 0, 1]
    rlen = list(range(1, 131)) + [40, 64, 7]
    rng = np.random.default_rng(6)
    q = rng.standard_normal((133, 9, 64)).astype(np.float32)
    for window, sinks in [(0, 0), (20, 2)]:
        o = gpu.allocate(q.shape, np.float32)
        paged_attention(cache.kv, gpu.to_device(q), i32(rlen), o, row_seq=i32(seqs),
                        window=window, sinks=sinks)
        want = attend(cache, q, seqs, rlen, window, sinks)
        assert head_error(o.to_numpy().astype(np.float64), want) < F32_TOL
    assert gpu.device_error() == 0


@pytest.mark.parametrize("D,P,dtype", [(128, 64, "bf16"), (64, 16, "bf16"), (64, 20, "bf16"),
                                       (64, 16, "f32")])
def test_attention_bad_indices_are_reported(D, P, dtype):
    """A page out of range makes its tokens invisible; lengths above the
    table's capacity are clamped; sequences out of range give zeros."""
    lens = [3 * P, 2 * P + 3, 5]
    cache = Cache(lens, 2, D, P, dtype, 7)
    q = np.random.default_rng(8).standard_normal((3, 4, D)).astype(np.float32)
    qd, o = gpu.to_device(q), gpu.allocate((3, 4, D), np.float32)
    good = attend(cache, q, [0, 1, 2], lens)
    for bad in (cache.kv.n_pages, -1, 2 ** 31 - 1):
        t = cache.table.copy()
        t[0, 1] = bad
        kv = PagedKV(cache.kv.k, cache.kv.v, i32(t))
        gpu.device_error(reset=True)
        paged_attention(kv, qd, i32(lens), o)
        got = o.to_numpy().astype(np.float64)
        assert gpu.device_error() == 32
        assert head_error(got[1:], good[1:]) < F32_TOL
        at = list(range(P)) + list(range(2 * P, 3 * P))
        k, v = cache.keys(0, at)
        for h in range(4):
            s = k[:, h // 2] @ q[0, h].astype(np.float64) * D ** -0.5
            w = np.exp(s - s.max())
            want = w @ v[:, h // 2] / w.sum()
            assert np.linalg.norm(got[0, h] - want) < F32_TOL * np.linalg.norm(want)
    gpu.device_error(reset=True)
    paged_attention(cache.kv, qd, i32([10 ** 9, -5, 5]), o)
    got = o.to_numpy().astype(np.float64)
    assert gpu.device_error() & 2      # clamped (row 0 covers all its pages)
    assert head_error(got[[0, 2]], good[[0, 2]]) < F32_TOL and (got[1] == 0).all()
    paged_attention(cache.kv, qd, i32(lens), o, row_seq=i32([0, 3, -1]))
    got = o.to_numpy().astype(np.float64)
    assert gpu.device_error() == 32
    assert head_error(got[:1], good[:1]) < F32_TOL and (got[1:] == 0).all()


@pytest.mark.parametrize("D,P,dtype", [(128, 64, "bf16"), (64, 16, "bf16"), (64, 16, "f32")])
def test_attention_extreme_scores(D, P, dtype):
    """Scores of +-1e4, equal scores, and NaN or infinite visible values."""
    lens = [200, 200, 200, 200]
    cache = Cache(lens, 1, D, P, dtype, 9)
    rng = np.random.default_rng(10)
    q = rng.standard_normal((4, 2, D)).astype(np.float32)
    q[0] *= 3000
    q[1] = 0
    o = gpu.allocate(q.shape, np.float32)
    paged_attention(cache.kv, gpu.to_device(q), i32(lens), o)
    got = o.to_numpy().astype(np.float64)
    want = attend(cache, q, range(4), lens)
    # score errors grow with the scores: 3000 times larger products
    assert head_error(got[:1], want[:1]) < 3000 * F32_TOL
    assert head_error(got[1:], want[1:]) < F32_TOL
    cache.k[cache.table[2, 1], 0, 3, 1] = np.nan
    cache.v[cache.table[3, 1], 0, 3, 1] = np.inf
    kv = PagedKV(up(cache.k, dtype), up(cache.v, dtype), i32(cache.table))
    paged_attention(kv, gpu.to_device(q), i32(lens), o)
    bad = o.to_numpy()
    assert np.isnan(bad[2]).all()
    assert (bad[3, :, 1] == np.inf).all() and np.isfinite(np.delete(bad[3], 1, 1)).all()
    assert (bad[:2] == got[:2].astype(np.float32)).all()


def test_attention_offsets_past_32_bits():
    """Pages whose element offsets pass 2^31, K and V of 4.3 GB each."""
    K, P, D = 8, 64, 128
    n = 2 ** 31 // (K * P * D) + 40
    k, v = gpu.allocate((n, K, P, D), "bfloat16"), gpu.allocate((n, K, P, D), "bfloat16")
    cache = Cache([250, 100], K, D, P, "bf16", 11, spare=0)
    m = len(cache.k)
    size = K * P * D * 2
    for big, small in ((k, cache.kv.k), (v, cache.kv.v)):
        gpu.copy_d2d(gpu.sub_view(big, (n - m) * size, (m, K, P, D)), small)
    table = np.where(cache.table < 0, -1, cache.table + n - m)
    q = np.random.default_rng(12).standard_normal((2, 24, D)).astype(np.float32)
    o = gpu.allocate(q.shape, np.float32)
    paged_attention(PagedKV(k, v, i32(table)), gpu.to_device(q), i32([250, 100]), o)
    want = attend(cache, q, [0, 1], [250, 100])
    assert head_error(o.to_numpy().astype(np.float64), want) < F32_TOL


def test_attention_of_a_table_near_its_largest():
    """Two sequences that may have 2^30 - 2^20 tokens; rows in more than one
    block of the kernel."""
    K, P, D, cols, R = 1, 1 << 20, 64, 1023, 600
    rng = np.random.default_rng(41)
    kv = [gpu.allocate((2, K, P, D), "bfloat16") for _ in range(2)]
    host = bf16(rng.standard_normal((2, 300, D)).astype(np.float32))   # page 1's first tokens
    for t, h in zip(kv, host):
        gpu.copy_d2d(gpu.sub_view(t, P * D * 2, (300, D)), gpu.to_device_bf16(h))
    table = np.full((2, cols), -1, np.int32)
    table[1, 0] = 1
    lens = rng.integers(0, 301, R)
    q = rng.standard_normal((R, 5, D)).astype(np.float32)
    o = gpu.allocate(q.shape, np.float32)
    paged_attention(PagedKV(*kv, i32(table)), gpu.to_device(q), i32(lens), o,
                    row_seq=i32(np.ones(R)))
    k, v = host.astype(np.float64)
    s = q.astype(np.float64) @ k.T / 8.0
    s[np.broadcast_to(np.arange(300) >= lens[:, None, None], s.shape)] = -np.inf
    w = np.exp(s - np.maximum(s.max(-1, keepdims=True), -1e30))
    want = w @ v / np.maximum(w.sum(-1, keepdims=True), 1e-30)
    assert head_error(o.to_numpy().astype(np.float64), want) < F32_TOL
    assert gpu.device_error() == 0


def test_attention_repeats_and_other_streams():
    """The same bits on every call, in a graph and on another stream."""
    from triton_llm import _lib
    import ctypes
    lens = [3000, 1, 777, 64]
    cache = Cache(lens, 8, 128, 64, "bf16", 13)
    q = gpu.to_device(np.random.default_rng(14).standard_normal((4, 24, 128))
                      .astype(np.float32))
    ld, o = i32(lens), gpu.allocate((4, 24, 128), np.float32)
    paged_attention(cache.kv, q, ld, o)
    first = o.to_numpy()
    for _ in range(20):
        paged_attention(cache.kv, q, ld, o)
    assert (o.to_numpy() == first).all()
    g = gpu.Graph()
    with g:
        paged_attention(cache.kv, q, ld, o)
    gpu.memset(o, 0)
    g.launch()
    assert (o.to_numpy() == first).all()
    s = ctypes.c_void_p()
    _lib.call("tllm_stream_create", ctypes.byref(s))
    with pytest.raises(ValueError, match="workspace"):
        paged_attention(cache.kv, q, ld, o, stream=s)
    gpu.memset(o, 0)
    gpu.synchronize()
    paged_attention(cache.kv, q, ld, o, stream=s, workspace=PagedWorkspace(4, 24, 8, 128))
    gpu.stream_synchronize(s)
    assert (o.to_numpy() == first).all()
    _lib.call("tllm_stream_destroy", s)


# -- append -----------------------------------------------------------------
def rotate(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    x = x.astype(np.float64).copy()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else \
        (slice(0, r // 2), slice(r // 2, r))
    u, w = x[..., a].copy(), x[..., b].copy()
    c, s = cos[:, None, :].astype(np.float64), sin[:, None, :].astype(np.float64)
    x[..., a], x[..., b] = u * c - w * s, w * c + u * s
    return x


def tables(n, r):
    ang = np.arange(n)[:, None] * 10000.0 ** (-np.arange(r // 2) / (r // 2))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,K,D,rot,P,blocked,slots_first", [
    (9, 3, 64, 64, 16, False, False), (24, 8, 128, 128, 64, True, False),
    (24, 8, 128, 64, 20, False, True), (4, 2, 96, 48, 16, False, False),
    (4, 1, 80, 20, 7, False, False), (3, 3, 18, 6, 4, False, False),
    (16, 2, 128, 0, 32, False, False), (2, 1, 32, 32, 1, True, True),
    (5, 5, 64, 2, 16, False, False)])
def test_append(H, K, D, rot, P, blocked, slots_first, interleaved, dtype):
    rng = np.random.default_rng(D + rot)
    seqs = np.array([2, 0, 0, 0, 3, 2, 1])
    pos = np.array([40, 0, 1, 2, 3 * P - 1, 41, P], np.int64)
    R, S, cols, n = len(pos), 4, 60 // P + 4, 300
    pages = rng.permutation(n)[:S * cols].reshape(S, cols).astype(np.int32)
    shape = (n, P, K, D) if slots_first else (n, K, P, D)
    k0 = bf16(rng.standard_normal(shape).astype(np.float32))
    v0 = bf16(rng.standard_normal(shape).astype(np.float32))
    kv = PagedKV(up(k0, dtype), up(v0, dtype), i32(pages), slots_first=slots_first)
    x = rng.standard_normal((R, H + 2 * K, D)).astype(np.float32)
    src = x
    if blocked:
        half = D // 2
        order = np.concatenate([np.r_[8 * b:8 * b + 8, half + 8 * b:half + 8 * b + 8]
                                for b in range(half // 8)])
        src = np.ascontiguousarray(x[..., order])
    cos, sin = tables(200, rot) if rot else (None, None)
    qo, lens = gpu.allocate((R, H, D), np.float32), gpu.zeros((S,), np.int32)
    gpu.device_error(reset=True)
    paged_append(kv, gpu.to_device(src.reshape(R, -1)), i32(pos), qo,
                 None if cos is None else gpu.to_device(cos),
                 None if sin is None else gpu.to_device(sin), n_head=H, row_seq=i32(seqs),
                 interleaved=interleaved, blocked=blocked, lens_out=lens)
    assert gpu.device_error() == 0
    turn = (lambda a: rotate(a, cos[pos], sin[pos], interleaved)) if rot else \
        (lambda a: a.astype(np.float64))
    wq, wk = turn(x[:, :H]), turn(x[:, H:H + K])
    norm = np.abs(x).max() * np.sqrt(2)
    got = qo.to_numpy().astype(np.float64)
    assert np.abs(got - wq).max() <= 3 * 2.0 ** -24 * norm
    assert (got[..., rot:] == x[:, :H, rot:]).all()
    kg, vg = gpu.to_host(kv.k), gpu.to_host(kv.v)
    kw, vw = k0.copy(), v0.copy()
    for r in range(R):
        p, s = pages[seqs[r], pos[r] // P], pos[r] % P
        at = (p, s) if slots_first else (p, slice(None), s)
        kr = kg[at].astype(np.float64)
        tol = 3 * 2.0 ** -24 * norm + (2.0 ** -8 * np.abs(wk[r]) if dtype == "bf16" else 0)
        assert (np.abs(kr - wk[r]) <= tol).all()
        kw[at] = kg[at]
        vw[at] = bf16(x[r, H + K:]) if dtype == "bf16" else x[r, H + K:]
    assert (kg == kw).all() and (vg == vw).all()     # nothing else is touched
    assert lens.to_numpy().tolist() == [3, P + 1, 42, 3 * P]


def test_append_many_rows():
    """72 MB of results (stored as streams), neighbouring pairs, half a head."""
    H, K, D, P, R = 24, 8, 128, 16, 3531
    rng = np.random.default_rng(9)
    x = rng.standard_normal((R, H + 2 * K, D), dtype=np.float32)
    pages = rng.permutation(R // P + 1).reshape(1, -1).astype(np.int32)
    zero = np.zeros((R // P + 1, K, P, D), np.float32)
    kv = PagedKV(up(zero, "bf16"), up(zero, "bf16"), i32(pages))
    cos, sin = tables(R, 64)
    qo, pos = gpu.allocate((R, H, D), np.float32), np.arange(R)
    paged_append(kv, gpu.to_device(x.reshape(R, -1)), i32(pos), qo, gpu.to_device(cos),
                 gpu.to_device(sin), n_head=H, row_seq=i32(np.zeros(R)), interleaved=True)
    norm = np.abs(x).max() * np.sqrt(2)
    want = rotate(x[:, :H + K], cos, sin, True)
    assert np.abs(qo.to_numpy() - want[:, :H]).max() <= 3 * 2.0 ** -24 * norm
    page, slot = pages[0, pos // P], pos % P
    k, v = gpu.to_host(kv.k)[page, :, slot], gpu.to_host(kv.v)[page, :, slot]
    assert (np.abs(k - want[:, H:]) <= 2.0 ** -8 * np.abs(want[:, H:]) + 3 * 2.0 ** -24
            * norm).all()
    assert (v == bf16(x[:, H + K:])).all()


def test_append_in_place_and_bad_rows():
    """q rotated in place; rows with a bad index are skipped and reported."""
    H, K, D, P, R = 4, 2, 64, 16, 6
    rng = np.random.default_rng(1)
    n = 8
    pages = np.array([[0, 1], [2, 3], [4, -1], [n, 6]], np.int32)
    zero = np.zeros((n, K, P, D), np.float32)
    kv = PagedKV(gpu.to_device(zero), gpu.to_device(zero), i32(pages))
    x = rng.standard_normal((R, H + 2 * K, D)).astype(np.float32)
    cos, sin = tables(30, D)
    seqs = [0, 1, 2, 3, 9, 1]
    pos = [3, 30, 20, 2, 1, 17]     # 30 is past the tables; seq 9 is none
    d = gpu.to_device(x.reshape(R, -1))
    gpu.device_error(reset=True)
    from triton_llm import _lib
    import ctypes
    r = _lib.PagedRowsStruct()
    at = d.data_ptr()
    r.q, r.k, r.v = at, at + H * D * 4, at + (H + K) * D * 4
    cd, sd, pd, qd = gpu.to_device(cos), gpu.to_device(sin), i32(pos), i32(seqs)
    r.q_out, r.row_pos, r.row_seq = at, pd.data_ptr(), qd.data_ptr()
    r.cos_t, r.sin_t, r.n_pos, r.rotary_dim = cd.data_ptr(), sd.data_ptr(), 30, D
    for f in ("q", "k", "v", "q_out"):
        setattr(r, f + "_row_stride", (H + 2 * K) * D)
        setattr(r, f + "_head_stride", D)
    r.rows, r.n_head = R, H
    _lib.call("tllm_paged_append", kv._ref, ctypes.addressof(r), None)
    assert gpu.device_error() == 32
    got = d.to_numpy().reshape(x.shape)
    ok = [0, 5]
    want = rotate(x[ok][:, :H], cos[[3, 17]], sin[[3, 17]], False)
    assert np.abs(got[ok][:, :H] - want).max() < 3 * 2.0 ** -24 * np.abs(x).max() * 1.5
    assert (got[1:5] == x[1:5]).all() and (got[:, H:] == x[:, H:]).all()
    k = kv.k.to_numpy()
    assert sorted(set(np.argwhere(k != 0)[:, 0])) == [0, 3]
    assert sorted(set(np.argwhere(k != 0)[:, 2])) == [1, 3]


@pytest.mark.parametrize("src_dtype,dtype", [("bf16", "bf16"), ("bf16", "f32"),
                                             ("f32", "bf16"), ("f32", "f32")])
def test_write_from_a_contiguous_cache(src_dtype, dtype):
    """Rows of a (sequence, head, slot) cache into pages, picked by row_src."""
    K, D, P, S = 3, 64, 16, 50
    rng = np.random.default_rng(2)
    ks = bf16(rng.standard_normal((2, K, S, D)).astype(np.float32))
    vs = bf16(rng.standard_normal((2, K, S, D)).astype(np.float32))
    zero = np.zeros((12, K, P, D), np.float32)
    pages = np.arange(12)[::-1].reshape(3, 4).astype(np.int32)
    kv = PagedKV(up(zero, dtype), up(zero, dtype), i32(pages))
    seq = np.r_[np.full(37, 0), np.full(50, 1)]
    pos = np.r_[np.arange(37), np.arange(50)]
    paged_write(kv, up(ks, src_dtype), up(vs, src_dtype), i32(pos), row_seq=i32(2 * seq),
                row_src=i32(seq * K * S + pos), row_stride=D, head_stride=S * D)
    for host, got in ((ks, gpu.to_host(kv.k)), (vs, gpu.to_host(kv.v))):
        want = zero.copy()
        for s, p in zip(seq, pos):
            want[pages[2 * s, p // P], :, p % P] = host[s, :, p]
        assert (got == want).all()


@pytest.mark.parametrize("P", [16, 7])
def test_write_skips_source_rows_out_of_range(P):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 2, 64)).astype(np.float32)
    zero = np.zeros((4, 2, P, 64), np.float32)
    kv = PagedKV(gpu.to_device(zero), gpu.to_device(zero), i32([[0, 1], [2, 3]]))
    gpu.device_error(reset=True)
    paged_write(kv, gpu.to_device(x), gpu.to_device(x), i32([0, 1, 2, 3]),
                row_seq=i32([0, 0, 1, 1]), row_src=i32([2, 3, -1, 0]))
    assert gpu.device_error() == 32
    want = zero.copy()
    want[0, :, 0], want[2, :, 3] = x[2], x[0]
    assert (kv.k.to_numpy() == want).all() and (kv.v.to_numpy() == want).all()


# -- page copies ------------------------------------------------------------
@pytest.mark.parametrize("dtype,shape,slots_first", [
    ("bf16", (4, 20, 3, 16, 64), False), ("f32", (2, 20, 8, 5, 128), False),
    ("bf16", (56, 30, 1, 64, 128), False), ("bf16", (3, 20, 16, 3, 64), True),
    ("bf16", (2, 20, 3, 7, 10), False), ("bf16", (2, 20, 3, 7, 9), False),
    ("f32", (1, 20, 1, 1, 1), False)])
@pytest.mark.parametrize("partial", [False, True])
def test_page_copy(dtype, shape, slots_first, partial):
    rng = np.random.default_rng(3)
    a = bf16(rng.standard_normal(shape).astype(np.float32))
    slots = shape[2] if slots_first else shape[3]
    src = np.array([1, 1, 2, -1, 7, 5, 6, 9])
    dst = np.array([10, 11, 12, 13, -1, 5, 17, 18])
    fill = rng.integers(0, slots + 1, len(src)) if partial else None
    d = up(a, dtype)
    gpu.device_error(reset=True)
    page_copy(d, i32(src), i32(dst), None if fill is None else i32(fill),
              slots_first=slots_first)
    want = a.copy()
    for i, (s, t) in enumerate(zip(src, dst)):
        if s < 0 or t < 0 or s == t:
            continue
        n = slots if fill is None else fill[i]
        at = (slice(None), slice(0, n)) if slots_first else \
            (slice(None), slice(None), slice(0, n))
        want[:, t][at] = a[:, s][at]
    assert (gpu.to_host(d) == want).all() and gpu.device_error() == 0


def test_page_copy_bad_entries_are_skipped():
    a = np.random.default_rng(4).standard_normal((2, 6, 2, 4, 8)).astype(np.float32)
    d = gpu.to_device(a)
    for src, dst, fill in [(6, 1, 4), (1, 6, 4), (1, 2, 5), (1, 2, -1)]:
        gpu.device_error(reset=True)
        page_copy(d, i32([src]), i32([dst]), i32([fill]))
        assert (d.to_numpy() == a).all() and gpu.device_error() == 32


# -- beam search ------------------------------------------------------------
def select(logits, scores, k, done=None, pad=0):
    """(scores, parents, tokens) in 64 bits, ties to the lowest index."""
    G, W = scores.shape
    V = logits.shape[1]
    x = logits.astype(np.float64).reshape(G, W, V)
    with np.errstate(all="ignore"):
        m = x.max(axis=2, keepdims=True)
        m0 = np.where(np.isfinite(m), m, 0)
        c = scores[:, :, None].astype(np.float64) + \
            (x - (m0 + np.log(np.exp(x - m0).sum(axis=2, keepdims=True))))
    c[np.isnan(c)] = -np.inf
    c[np.isposinf(scores)] = -np.inf
    if done is not None:
        for g, b in np.argwhere(done.reshape(G, W) != 0):
            c[g, b] = -np.inf
            c[g, b, pad] = scores[g, b]
    c = c.reshape(G, W * V)
    at = np.argsort(-c, axis=1, kind="stable")[:, :k]
    return np.take_along_axis(c, at, 1), at // V, at % V


def run_select(logits, scores, k, done=None, pad=0, ld=None):
    G = scores.shape[0]
    s, p, t = (gpu.allocate((G, k), d) for d in (np.float32, np.int32, np.int32))
    beam_select(gpu.to_device(logits), gpu.to_device(scores), s, p, t,
                done=None if done is None else i32(done), pad_token=pad)
    return s.to_numpy(), p.to_numpy(), t.to_numpy()


@pytest.mark.parametrize("G,W,V,k", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 6),
                                     (1, 4, 1000, 4), (3, 5, 4096, 10), (2, 8, 4097, 16),
                                     (1, 32, 3001, 64), (16, 8, 50257, 8),
                                     (1, 4, 128256, 64), (4, 2, 131, 64)])
def test_beam_select(G, W, V, k):
    """The gaps between the best scores are far above fp32 rounding, so the
    choice is exact; scores are a sum of three fp32 terms of size < 64: off
    by at most 2^-17 of rounding and the logarithm's own."""
    rng = np.random.default_rng(V)
    logits = (rng.standard_normal((G * W, V)) * 3).astype(np.float32)
    scores = (-rng.random((G, W)) * 30).astype(np.float32)
    done = (rng.random((G, W)) < 0.25).astype(np.int32)
    for d in (None, done):
        s, p, t = run_select(logits, scores, k, d, V - 1)
        ws, wp, wt = select(logits, scores, k, d, V - 1)
        fine = np.isfinite(ws)
        assert (np.isfinite(s) == fine).all() and (s[~fine] == ws[~fine]).all()
        assert np.abs(s[fine] - ws[fine]).max() < 2.0 ** -16
        assert (p == wp).all() and (t == wt).all()


def test_beam_select_ties_and_special_values():
    V = 5000
    inf = np.float32(np.inf)
    # all equal: the lowest beams and tokens
    s, p, t = run_select(np.zeros((3, V), np.float32), np.zeros((1, 3), np.float32), 6)
    assert p.tolist() == [[0] * 6] and t.tolist() == [list(range(6))]
    # equal logits far apart, -0 and +0 alike
    x = np.full((2, V), -9, np.float32)
    x[:, [4999, 17, 2048]] = [0.0, -0.0, 0.0]
    s, p, t = run_select(x, np.zeros((1, 2), np.float32), 6)
    assert p.tolist() == [[0, 0, 0, 1, 1, 1]]
    assert t.tolist() == [[17, 2048, 4999] * 2]
    # the first step: one live beam
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, V)).astype(np.float32)
    live = np.array([[0, -inf, -inf, -inf]], np.float32)
    s, p, t = run_select(x, live, 4)
    assert (p == 0).all() and (t == select(x, live, 4)[2]).all()
    # masked tokens, rows that are all masked, NaN, infinities
    x[0, 7:] = -inf
    x[1] = -inf
    x[2, 3] = np.nan
    x[3, 3] = inf
    sc = np.zeros((1, 4), np.float32)
    s, p, t = run_select(x, sc, 12)
    ws, wp, wt = select(x, sc, 12)
    assert (p == wp).all() and (t == wt).all()
    assert (np.isfinite(s) == np.isfinite(ws)).all() and np.isfinite(s).sum() == 7
    # beams without a score, of +inf and NaN
    x = rng.standard_normal((4, V)).astype(np.float32)
    sc = np.array([[np.nan, inf, -inf, -3]], np.float32)
    s, p, t = run_select(x, sc, 5)
    assert (p == 3).all() and (t == select(x, sc, 5)[2]).all()


def reorder(parents, lens, table, P):
    G, W = parents.shape
    out = table.copy()
    src, dst, fill = (np.full(G * W, x, np.int32) for x in (-1, -1, 0))
    for g in range(G):
        c, f = divmod(int(lens[g * W]), P)
        old = table[g * W:(g + 1) * W]
        new = old.copy()
        new[:, :c] = old[parents[g], :c]
        if f:
            seen, ends = set(), [b for b in range(W) if b not in parents[g]]
            for i, b in enumerate(parents[g]):
                take = b if b not in seen else ends.pop(0)
                seen.add(b)
                new[i, c] = old[take, c]
                src[g * W + i], dst[g * W + i] = old[b, c], old[take, c]
                fill[g * W + i] = f
        out[g * W:(g + 1) * W] = new
    return out, src, dst, fill


@pytest.mark.parametrize("G,W,C,P", [(1, 1, 1, 4), (2, 4, 5, 16), (5, 8, 40, 1),
                                     (3, 32, 300, 64), (16, 5, 33, 7)])
@pytest.mark.parametrize("in_place", [False, True])
def test_beam_reorder(G, W, C, P, in_place):
    rng = np.random.default_rng(C)
    for step in range(4):
        table = rng.permutation(G * W * C).reshape(G * W, C).astype(np.int32)
        parents = rng.integers(0, W, (G, W)).astype(np.int32)
        if step == 1:
            parents[:] = np.arange(W)
        lens = np.repeat(rng.integers(0, C * P + 1, G), W).astype(np.int32)
        if step == 2:
            lens[:] = lens // P * P
        tin = i32(table)
        tout = tin if in_place else gpu.allocate((G * W, C), np.int32)
        c = [gpu.allocate((G * W,), np.int32) for _ in range(3)]
        gpu.device_error(reset=True)
        beam_reorder(i32(parents), i32(lens), tin, tout, *c, page_size=P)
        want = reorder(parents, lens, table, P)
        for got, w in zip([tout] + c, want):
            assert (got.to_numpy() == w).all()
        assert gpu.device_error() == 0


def test_beam_reorder_bad_indices():
    table = np.arange(12).reshape(4, 3).astype(np.int32)
    for parents, lens in [([[0, 2], [1, 0]], [5] * 4), ([[0, -1], [1, 0]], [5] * 4),
                          ([[0, 0], [1, 0]], [13, 13, 5, 5]),
                          ([[0, 0], [1, 0]], [-1, -1, 5, 5])]:
        tout = gpu.allocate((4, 3), np.int32)
        c = [gpu.allocate((4,), np.int32) for _ in range(3)]
        gpu.device_error(reset=True)
        beam_reorder(i32(parents), i32(lens), i32(table), tout, *c, page_size=4)
        assert gpu.device_error() == 32
        want = reorder(np.array([[0, 1], [1, 0]]), np.array([0, 0, 5, 5]), table, 4)
        assert (tout.to_numpy() == want[0]).all()
        assert (c[0].to_numpy()[:2] == -1).all() and (c[0].to_numpy()[2:] == want[1][2:]).all()


def test_operators_take_torch_tensors():
    """CUDA tensors of torch, with strides, beside DeviceTensors."""
    torch = pytest.importorskip("torch")
    lens = [100, 33]
    cache = Cache(lens, 2, 64, 16, "bf16", 15)
    both = torch.stack([torch.from_numpy(cache.k), torch.from_numpy(cache.v)], 1)
    both = both.bfloat16().cuda()          # K and V interleaved page by page
    table = torch.from_numpy(cache.table).cuda()
    wide = torch.randn(2, 6, 64, device="cuda")
    q = wide[:, 1:5]                       # rows 6 * 64 apart
    out = torch.empty(2, 4, 64, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    paged_attention(PagedKV(both[:, 0], both[:, 1], table), q, n, out)
    gpu.synchronize()
    want = attend(cache, q.cpu().numpy(), [0, 1], lens)
    assert head_error(out.cpu().numpy().astype(np.float64), want) < F32_TOL


@pytest.mark.parametrize("V,k", [(40000, 8), (40000, 64), (128256, 16), (9000, 33)])
def test_beam_select_clustered_values(V, k):
    """Large values where they crowd one thread's, warp's or step's share: runs,
    strides of the kernel's step and sorted rows; equal values across them."""
    rng = np.random.default_rng(V + k)
    base = rng.standard_normal((8, V)).astype(np.float32)
    rows = [np.sort(base[0]), np.sort(base[1])[::-1].copy()]
    for stride in (4096, 1024, 128, 512):
        x = base[len(rows)].copy()
        at = np.arange(stride // 2, V, stride)
        x[at] = 20 + rng.permutation(len(at)).astype(np.float32) / 8
        rows.append(x)
    x = base[6].copy()
    x[777:777 + 300] = 9 + np.arange(300, dtype=np.float32) / 16
    rows.append(x)
    x = np.round(base[7] * 2) / 2           # many equal ones
    x[:V // 2] = -np.inf
    rows.append(x)
    logits = np.stack(rows)
    # one row a group, so that every row's own order shows
    s, p, t = run_select(logits, np.zeros((8, 1), np.float32), k)
    ws, wp, wt = select(logits, np.zeros((8, 1), np.float32), k)
    assert np.abs(s - ws).max() < 2.0 ** -14
    assert (t == wt).all()
