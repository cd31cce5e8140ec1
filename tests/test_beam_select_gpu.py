"""Beam selection on a B200 where its numbers and its paths are hardest: many
steps of one thread, large logits, masks of the type's lowest value, scores that
collapse in fp32, row strides.

Oracle: base + ((x - max) - log(sum exp(x - max))) in 64 bits, which keeps the
logarithm beside a maximum of 1e38 too. Tolerance 2^-16 for scores below 64: a
sum of up to 160 fp32 additions of positive terms is off by less than 160 * 2^-24
= 2^-16.7 of itself, a term by 2^-22 of the exponential and 15 * 2^-23 of its
argument (terms further below the maximum do not count), the subtraction and the
logarithm by 2^-21. Scores near the type's lowest value are off by their own
rounding, 2^-23.
"""

from __future__ import annotations

import numpy as np
import pytest

from triton_llm import gpu
from triton_llm.kernels import beam_select

pytestmark = pytest.mark.gpu

LOWEST = np.finfo(np.float32).min
# more rows than a GPU has places for CTAs: a row is not cut into parts, and a
# thread reads a step of 4096 logits of it after another
MANY = 600


def candidates(logits, scores, done=None, pad=0):
    """(groups, beams * vocab) candidate scores in 64 bits."""
    G, W = scores.shape
    x = logits.astype(np.float64).reshape(G, W, -1)
    m = x.max(axis=2, keepdims=True)
    lp = (x - m) - np.log(np.exp(x - m).sum(axis=2, keepdims=True))
    c = scores[:, :, None].astype(np.float64) + lp
    if done is not None:
        for g, b in np.argwhere(done != 0):
            c[g, b] = -np.inf
            c[g, b, pad] = scores[g, b]
    return c.reshape(G, -1)


def best(c, k, vocab):
    """The k best, ties to the lowest index."""
    at = np.argsort(-c, axis=1, kind="stable")[:, :k]
    return np.take_along_axis(c, at, 1), at // vocab, at % vocab


def run(logits, scores, k, done=None, pad=0):
    G = scores.shape[0]
    s, p, t = (gpu.allocate((G, k), d) for d in (np.float32, np.int32, np.int32))
    beam_select(logits if hasattr(logits, "data_ptr") else gpu.to_device(logits),
                gpu.to_device(scores), s, p, t,
                done=None if done is None else gpu.to_device(done.astype(np.int32)),
                pad_token=pad)
    return s.to_numpy(), p.to_numpy(), t.to_numpy()


def many(rows):
    """The rows again and again, MANY of them."""
    return np.ascontiguousarray(np.resize(rows, (MANY, rows.shape[1])))


@pytest.mark.parametrize("V", [128256, 50257])
def test_large_logits_in_many_steps(V):
    """32 (or 13) steps a thread: the running sum keeps its precision whatever
    the logits' size."""
    rng = np.random.default_rng(V)
    rows = (rng.standard_normal((8, V)) * 3).astype(np.float32)
    rows += np.array([0, 10, -20, 100, -100, 1000, -1000, 4000], np.float32)[:, None]
    zero = np.zeros((MANY, 1), np.float32)
    s, _, t = run(many(rows), zero, 8)
    ws, _, wt = best(candidates(rows, zero[:8]), 8, V)
    assert (t == np.resize(wt, t.shape)).all()
    assert np.abs(s - np.resize(ws, s.shape)).max() < 2.0 ** -16


def masked_rows(V):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((10, V)).astype(np.float32)
    x[0, :V // 2] = LOWEST               # a range of tokens, whole steps of it
    x[1, 1:] = LOWEST                    # all but one
    x[2, :-1] = LOWEST
    x[3, ::2] = LOWEST
    x[4] = LOWEST                        # all: the tokens are equally likely
    x[5, :] = LOWEST / 2
    x[5, 77] = LOWEST / 4
    x[6] = -LOWEST                       # the same at the other end
    x[7, 100:200] = -LOWEST
    x[8, :] = LOWEST
    x[8, 9:V - 9] = -np.inf              # both kinds of mask
    x[9, 17:4500] = LOWEST
    return x


@pytest.mark.parametrize("rows", [10, MANY])
@pytest.mark.parametrize("V,k", [(20000, 8), (20002, 64), (9001, 1)])
def test_masks_of_the_lowest_value(rows, V, k):
    """Finite logits whatever their size: masks of the type's lowest value on
    some, most and all tokens of a row."""
    x = masked_rows(V)
    with np.errstate(all="ignore"):
        ws, _, wt = best(candidates(x, np.zeros((10, 1), np.float32)), k, V)
    s, _, t = run(many(x) if rows == MANY else x, np.zeros((rows, 1), np.float32), k)
    ws, wt = np.resize(ws, s.shape), np.resize(wt, t.shape)
    assert (t == wt).all()
    fine = np.isfinite(ws)
    assert (s[~fine] == ws[~fine]).all()
    assert (np.abs(s[fine] - ws[fine]) <= 2.0 ** -16 + 2.0 ** -22 * np.abs(ws[fine])).all()


def test_a_masked_beam_beside_others():
    """A beam whose tokens are all masked alike has its 1 / vocab candidates
    among the other beams'."""
    V = 9000
    x = np.random.default_rng(4).standard_normal((4, V)).astype(np.float32) * 4
    x[2] = LOWEST
    scores = np.array([[-9, -30, 0, -5]], np.float32)
    s, p, t = run(x, scores, 12)
    ws, wp, wt = best(candidates(x, scores), 12, V)
    assert (p == wp).all() and (t == wt).all() and (wp == 2).any() and (wp != 2).any()
    assert np.abs(s - ws).max() < 2.0 ** -16


def rounded(c):
    """Candidates as the fp32 scores that they have, where these do not hang on
    the last bits of the logarithm: every one is further than 2^-13 of a unit
    from the middle of two."""
    s = c.astype(np.float32)
    unit = np.spacing(np.abs(s.max()))
    off = np.abs(c / unit - np.floor(c / unit) - 0.5)
    assert (off[np.isfinite(c)] > 2.0 ** -13).all()
    return s.astype(np.float64)


def best_of_equal(s, logits, k, vocab):
    """The k best by fp32 score, beam, logit and token, in this order."""
    x = logits.astype(np.float64).reshape(s.shape)
    n = np.arange(s.shape[1])
    at = np.stack([np.lexsort((n, -x[g], n // vocab, -s[g])) for g in range(len(s))])[:, :k]
    return np.take_along_axis(s, at, 1), at // vocab, at % vocab


@pytest.mark.parametrize("rows", ["few", "many"])
@pytest.mark.parametrize("V,W,k", [(20000, 1, 1), (20000, 1, 8), (5000, 4, 7), (12289, 3, 64),
                                   (40000, 2, 33)])
def test_equal_scores_of_unequal_logits(rows, V, W, k):
    """Beams so unlikely that many logits give the same fp32 score: one order of
    all candidates, by score, beam, logit and token, at the end of a part's list
    as among the listed ones."""
    rng = np.random.default_rng(V + k)
    x = rng.standard_normal((W, V)).astype(np.float32)
    x = np.round(x * 32) / 32
    base = np.full((1, W), -2.0 ** 20, np.float32)       # scores in units of 1/8
    base[0, W // 2] -= 1
    ws, wp, wt = best_of_equal(rounded(candidates(x, base)), x, k, V)
    assert (ws[0, 1:] == ws[0, :-1]).any() or k == 1
    G = 1 if rows == "few" else -(-MANY // W)
    s, p, t = run(np.tile(x, (G, 1)), np.tile(base, (G, 1)), k)
    assert (p == wp).all() and (t == wt).all() and (s == ws).all()


def test_scores_that_all_collapse():
    """All candidates of a beam equal (a score of -1e30): its largest logits, of
    the lowest beams; finished beams and masked tokens in their places."""
    V, k = 30000, 40
    x = np.random.default_rng(8).standard_normal((4, V)).astype(np.float32)
    x[1, :17] = -np.inf
    x[1, 19:] = LOWEST
    scores = np.array([[-2e30, -1e30, -1e30, -1e30]], np.float32)
    order = np.argsort(-x, axis=1, kind="stable")
    s, p, t = run(x, scores, k)
    # (two tokens at -1e30; LOWEST less the maximum is far below)
    assert p[0].tolist() == [1, 1] + [2] * (k - 2) and (s == np.float32(-1e30)).all()
    assert t[0].tolist() == order[1, :2].tolist() + order[2, :k - 2].tolist()
    done = np.array([[0, 1, 0, 0]])
    s, p, t = run(x, scores, k, done, V - 1)
    assert p[0].tolist() == [1] + [2] * (k - 1)
    assert t[0].tolist() == [V - 1] + order[2, :k - 1].tolist()
    x[1] = -np.inf                       # fewer than k candidates in all
    x[1, [5, 50, 500]] = [1, 3, 2]
    s, p, t = run(x[1:2], scores[:, 1:2], 6)
    assert t[0].tolist() == [50, 500, 5, 0, 1, 2]
    assert (s[0, :3] == np.float32(-1e30)).all() and (s[0, 3:] == -np.inf).all()


def crowded(V, lanes, kVec=True):
    """Rows whose large values all lie in the shares of a few threads, in every
    step of 4096 logits; the largest in the last ones."""
    rng = np.random.default_rng(V + lanes)
    at = np.arange(V)
    warp, inner = at % 4096 // 512, at % 512
    lane = inner % 128 // 4 if kVec else inner % 32
    x = rng.standard_normal((6, V)).astype(np.float32)
    for r in range(6):
        mine = np.isin(warp * 32 + lane, rng.choice(256, lanes, replace=False))
        n = int(mine.sum())
        large = 10 + rng.permutation(n).astype(np.float32) / 1024
        x[r, mine] = [np.sort(large), np.sort(large)[::-1], large, np.round(large * 4) / 4,
                      np.full(n, 11, np.float32), large][r]
    x[5, ::3] = -np.inf
    return x


@pytest.mark.parametrize("lanes", [1, 3, 20])
@pytest.mark.parametrize("V,k", [(40000, 1), (40000, 8), (40001, 64), (24576, 64)])
def test_values_crowded_into_few_threads(V, k, lanes):
    """A thread's third and later steps hold the best values (they are read
    again), and with 20 such threads more values pass the bound than the list
    holds (k rounds over all of them)."""
    x = crowded(V, lanes, V % 4 == 0)
    zero = np.zeros((MANY, 1), np.float32)
    s, _, t = run(many(x), zero, k)
    # (equal logits are equal scores; unequal ones are 2^-10 apart)
    ws, _, wt = best(candidates(x, zero[:6]), k, V)
    assert (t == np.resize(wt, t.shape)).all()
    assert np.abs(s - np.resize(ws, s.shape)).max() < 2.0 ** -16


@pytest.mark.parametrize("V,ld", [(5000, 5004), (5000, 5001), (3, 8), (128256, 128300)])
@pytest.mark.parametrize("G,W", [(1, 4), (3, 2), (75, 8)])
def test_rows_wider_than_the_vocabulary(V, ld, G, W):
    """Logits with a row stride above the vocabulary, whose rest is NaN."""
    torch = pytest.importorskip("torch")
    if G * W * ld > 1 << 25:
        G, W = 4, 2
    rng = np.random.default_rng(ld)
    x = (rng.standard_normal((G * W, V)) * 3).astype(np.float32)
    scores = (-rng.random((G, W)) * 30).astype(np.float32)
    wide = torch.full((G * W, ld), float("nan"))
    wide[:, :V] = torch.from_numpy(x)
    wide = wide.cuda()
    torch.cuda.synchronize()
    k = min(V, 5)
    s, p, t = run(wide[:, :V], scores, k)
    ws, wp, wt = best(candidates(x, scores), k, V)
    assert (p == wp).all() and (t == wt).all()
    assert np.abs(s - ws).max() < 2.0 ** -16
