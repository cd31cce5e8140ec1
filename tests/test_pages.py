"""Host-side accounting of pages, and the scaled rotary tables (CPU)."""

from __future__ import annotations

import numpy as np
import pytest

from triton_llm.kernels import precompute_cos_sin, scaled_cos_sin
from triton_llm.pages import PagePool


def test_take_share_release():
    p = PagePool(6)
    a = p.take(3)
    assert a.tolist() == [0, 1, 2] and p.used == 3 and p.free == 3
    p.share(a[:2])
    p.release(a)
    assert p.used == 2 and p.users.tolist() == [1, 1, 0, 0, 0, 0]
    assert p.take(2).tolist() == [2, 3]          # the lowest free ones
    p.release([0, 1, 2, 3])
    assert p.used == 0 and p.take(0).size == 0
    b = p.take(1)
    p.share([b[0], b[0]])
    p.release([b[0], b[0], b[0]])
    assert p.free == 6


def test_refusals_change_nothing():
    p = PagePool(4)
    a = p.take(3)
    with pytest.raises(RuntimeError, match="out of pages"):
        p.take(2)
    for bad in ([4], [-1]):
        with pytest.raises(ValueError, match="not all in"):
            p.release(bad)
    with pytest.raises(ValueError, match="are free"):
        p.share([3])
    with pytest.raises(ValueError, match="more often"):
        p.release([a[0], a[0]])
    with pytest.raises(ValueError):
        p.take(-1)
    with pytest.raises(ValueError):
        PagePool(-1)
    assert p.used == 3 and p.users.tolist() == [1, 1, 1, 0]


@pytest.mark.parametrize("seed", range(5))
def test_compact(seed):
    rng = np.random.default_rng(seed)
    p = PagePool(40)
    held = p.take(int(rng.integers(1, 40)))
    p.share(rng.choice(held, len(held) // 2, replace=False))
    drop = rng.choice(held, len(held) // 3, replace=False)
    for page in drop:
        p.release([page] * int(p.users[page]))
    keep = np.setdiff1d(held, drop)
    content = {int(x): (int(x), int(p.users[x])) for x in keep}
    src, dst, where = p.compact()
    assert not set(src) & set(dst) and len(src) == len(dst)
    assert sorted(where[keep].tolist()) == list(range(len(keep)))
    assert (where[src] == dst).all()
    for x, (_, users) in content.items():
        assert p.users[where[x]] == users
    assert p.used == len(keep) and p.take(p.free).tolist() == list(range(len(keep), 40))


def test_scaled_tables():
    """Against frequencies written down pair by pair in 64 bits."""
    n, d, theta = 300, 32, 10000.0
    c0, s0 = scaled_cos_sin(n, d, theta)
    # the plain tables form their angles in fp32: off by 2^-24 of 300 radians
    c1, s1 = precompute_cos_sin(n, d, theta)
    assert max(np.abs(c0 - c1).max(), np.abs(s0 - s1).max()) < 300 * 2.0 ** -22

    def check(scaling, freqs, size=1.0):
        c, s = scaled_cos_sin(n, d, theta, scaling)
        ang = np.arange(n)[:, None] * np.array(freqs)
        assert np.abs(c - size * np.cos(ang)).max() < 1e-6
        assert np.abs(s - size * np.sin(ang)).max() < 1e-6

    f = [theta ** (-2 * i / d) for i in range(d // 2)]
    check({"type": "linear", "factor": 4.0}, [x / 4 for x in f])
    base = theta * 4.0 ** (d / (d - 2))
    check({"rope_type": "ntk", "factor": 4.0}, [base ** (-2 * i / d) for i in range(d // 2)])
    orig, lo, hi = 128, 1.0, 4.0
    out = []
    for x in f:
        turns = orig * x / (2 * np.pi)
        keep = min(max((turns - lo) / (hi - lo), 0.0), 1.0)
        out.append(x * keep + x / 8 * (1 - keep))
    check({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": lo,
           "high_freq_factor": hi, "original_max_position_embeddings": orig}, out)
    assert out[0] == f[0] and out[-1] == f[-1] / 8
    lo_i = max(np.floor(d * np.log(orig / (32 * 2 * np.pi)) / (2 * np.log(theta))), 0)
    hi_i = min(np.ceil(d * np.log(orig / (2 * np.pi)) / (2 * np.log(theta))), d - 1)
    out = []
    for i, x in enumerate(f):
        keep = 1 - min(max((i - lo_i) / (hi_i - lo_i), 0.0), 1.0)
        out.append(x * keep + x / 4 * (1 - keep))
    check({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": orig},
          out, 0.1 * np.log(4.0) + 1)


@pytest.mark.parametrize("kw", [
    dict(scaling={"type": "linear"}), dict(scaling={"type": "linear", "factor": 0.5}),
    dict(scaling={"type": "sideways", "factor": 2}), dict(scaling={"type": "yarn", "factor": 2}),
    dict(scaling={"rope_type": "llama3", "factor": 2, "low_freq_factor": 4,
                  "high_freq_factor": 4, "original_max_position_embeddings": 64}),
    dict(d_k=31), dict(max_seq_len=0), dict(theta=0)])
def test_scaled_table_refusals(kw):
    with pytest.raises(ValueError):
        scaled_cos_sin(**dict(dict(max_seq_len=8, d_k=32), **kw))
