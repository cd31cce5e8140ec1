"""Models over a paged cache on a B200: against the same models over the
contiguous cache, and beam search against a plain search with the oracle.

Tolerances: both caches hold the same bf16 (or fp32) keys and values; q, the
attention's sums and its outputs differ by fp32 rounding (4e-6 of a value, see
test_paged_gpu), rounded to 2^-16 operand planes with bf16 weights, and pass
through two layers: logits within 1e-4 of their largest, as the parity bars of
test_models_gpu for fp32-like arithmetic.
"""

from __future__ import annotations

import numpy as np
import pytest

import inputs
from oracle import models as omodels

pytestmark = pytest.mark.gpu


def model(shape=inputs.SMOL_TINY, dtype=None, seed=42, weights=None, **kw):
    from smollm2_triton import SmolLM2Config, SmolLM2ForCausalLM
    w = weights or inputs.llama_weights_legacy(shape, seed)
    return SmolLM2ForCausalLM(SmolLM2Config(**shape.config_kwargs()), w, dtype=dtype, **kw), w


@pytest.fixture(autouse=True)
def no_device_errors():
    from triton_llm import gpu
    gpu.device_error(reset=True)
    yield
    assert gpu.device_error(reset=True) == 0


def prompts_of(shape, lens, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, shape.vocab_size, n).astype(np.int32) for n in lens]


def run(sess, prompts, steps):
    """Logits of the prompts' last tokens and of every greedy step."""
    out = [sess.prefill(prompts)]
    for _ in range(steps):
        sess.step()
        out.append(sess.logits.to_numpy()[:len(prompts)])
    return np.stack(out)


@pytest.mark.parametrize("dtype,P", [("float32", 5), ("float32", 64), ("bfloat16", 16),
                                     ("bfloat16", 7)])
def test_paged_session_equals_contiguous(dtype, P):
    from smollm2_triton.engine import LlamaSession
    from smollm2_triton.paged import PagedSession
    m, _ = model(dtype=dtype)
    m._init_gpu_weights()
    prompts = prompts_of(inputs.SMOL_TINY, [3, 40, 17])
    want = run(LlamaSession(m.dev, 3, 80), prompts, 30)
    for graph in (False, True):
        s = PagedSession(m.dev, 3, 80, page_size=P)
        if graph:
            s.prefill(prompts)
            s.capture()
        got = run(s, prompts, 30)
        assert np.abs(got - want).max() < 1e-4 * np.abs(want).max()
        assert (got.argmax(-1) == want.argmax(-1)).all()


@pytest.mark.parametrize("act", ["split", "bfloat16"])
def test_paged_llama3b_slice(act):
    """Llama-3.2-3B geometry (24 / 8 heads of 128), two layers, bf16."""
    from smollm2_triton.engine import LlamaSession, LlamaWeights
    from smollm2_triton.paged import PagedSession
    from smollm2_triton import SmolLM2Config
    shape = inputs.LLAMA3B_2L
    w = LlamaWeights(SmolLM2Config(**shape.config_kwargs()), dtype="bfloat16", seed=3)
    prompts = prompts_of(shape, [100, 300])
    want = run(LlamaSession(w, 2, 400, act_dtype=act), prompts, 8)
    got = run(PagedSession(w, 2, 400, page_size=64, act_dtype=act), prompts, 8)
    # one bf16 operand plane rounds at 2^-9: values that differ in their last
    # fp32 bits may round apart
    tol = 1e-4 if act == "split" else 2e-2
    assert np.abs(got - want).max() < tol * np.abs(want).max()


def test_generate_paged_equals_generate_batch():
    m, _ = model(dtype="bfloat16")
    prompts = prompts_of(inputs.SMOL_TINY, [9, 33, 1])
    want = m.generate_batch(prompts, max_new_tokens=40)
    for kw in (dict(), dict(page_size=16, use_graph=False), dict(window=512, sinks=4)):
        got = m.generate_paged(prompts, max_new_tokens=40, **kw)
        for a, b in zip(got, want):
            assert a.tolist() == b.tolist()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_window_steps_equal_window_prefill(dtype):
    """With a window, decoding token by token over freed pages gives what a
    prefill of the same tokens gives; and the window matters."""
    from smollm2_triton.paged import PagedSession
    m, _ = model(dtype=dtype)
    m._init_gpu_weights()
    ids = prompts_of(inputs.SMOL_TINY, [70])[0]
    kw = dict(page_size=8, window=20, sinks=3)
    s = PagedSession(m.dev, 1, 80, **kw)
    rows = [s.prefill([ids[:10]])[0]]
    peak = 0
    for t in range(10, 69):
        s.ids.from_numpy(ids[t:t + 1])
        s.decode_step(sample=True)
        rows.append(s.logits.to_numpy()[0])
        peak = max(peak, s.pool.used)
    assert peak <= 1 + 20 // 8 + 2          # sinks' page, the window's, one ahead
    full = PagedSession(m.dev, 1, 80, **kw).prefill([ids], all_logits=True)
    scale = np.abs(full).max()
    for t, row in zip(range(9, 69), rows):
        if t == 9:
            continue
        assert np.abs(row - full[t]).max() < 1e-4 * scale
    open_ = PagedSession(m.dev, 1, 80, page_size=8).prefill([ids], all_logits=True)
    assert np.abs(open_[:20] - full[:20]).max() < 1e-4 * scale
    assert np.abs(open_[60] - full[60]).max() > 1e-3 * scale


def test_fork_compact_release():
    from smollm2_triton.paged import PagedSession
    m, _ = model(dtype="bfloat16")
    m._init_gpu_weights()
    prompts = prompts_of(inputs.SMOL_TINY, [21, 50])
    alone = PagedSession(m.dev, 2, 120, page_size=8)
    want = run(alone, prompts, 40)[:, 0]
    s = PagedSession(m.dev, 4, 120, page_size=8, n_pages=40)
    s.prefill(prompts, slots=[2, 0])
    for _ in range(5):
        s.step()
    s.fork(2, [3, 1])                       # shares 3 full pages, copies one
    assert s.pool.users.max() == 3
    s.release([0])
    assert s.compact() > 0
    for step in range(5, 40):
        s.step()
        got = s.logits.to_numpy()[[2, 3, 1]]
        assert np.abs(got - want[step + 1]).max() < 1e-4 * np.abs(want).max()
        if step == 20:
            s.compact()
    s.release([2, 3])
    s.release([1])
    assert s.pool.used == 0
    for _ in range(20):                     # idle slots take none
        s.step()
    assert s.pool.used == 0


def test_slots_and_page_limits():
    from smollm2_triton.paged import PagedSession
    m, _ = model(dtype="bfloat16")
    m._init_gpu_weights()
    p = prompts_of(inputs.SMOL_TINY, [30])[0]
    s = PagedSession(m.dev, 2, 64, page_size=16, n_pages=3)
    s.prefill([p], slots=[0])
    with pytest.raises(RuntimeError, match="out of pages"):
        s.prefill([p], slots=[1])
    for _ in range(18):                     # up to position 48 = 3 pages of 16
        s.step()
    with pytest.raises(RuntimeError, match="out of pages"):
        s.step()
    for kw in (dict(page_size=0), dict(sinks=2), dict(window=-1)):
        with pytest.raises(ValueError):
            PagedSession(m.dev, 2, 64, **kw)
    with pytest.raises(ValueError, match="fork"):
        s.fork(1, [0])
    with pytest.raises(ValueError, match="fork"):
        s.fork(0, [2])
    with pytest.raises(ValueError, match="slots"):
        s.release([-1])


def test_sequences_survive_when_pages_run_out():
    """A prompt, a fork or a step that finds too few pages leaves the other
    sequences as they were: they go on as if it had not been tried."""
    from smollm2_triton.paged import PagedSession
    m, _ = model(dtype="bfloat16")
    m._init_gpu_weights()
    a, b = prompts_of(inputs.SMOL_TINY, [21, 30])
    want = run(PagedSession(m.dev, 1, 96, page_size=8), [a], 30)[:, 0]
    s = PagedSession(m.dev, 4, 96, page_size=8, n_pages=8)
    got = [s.prefill([a], slots=[1])[0]]    # 3 pages

    def step(n):
        for _ in range(n):
            s.step()
            got.append(s.logits.to_numpy()[1])
    s.prefill([b], slots=[2])               # 4 pages, 1 is left
    step(1)
    with pytest.raises(RuntimeError, match="out of pages"):
        s.fork(1, [0, 3])                   # needs two
    with pytest.raises(RuntimeError, match="out of pages"):
        s.prefill([b], slots=[0])
    step(1)                                 # (slot 2 is at 32 = 4 pages, slot 1 at 23)
    s.fork(1, [3])                          # shares 2 pages, the last free one is its own
    assert s.pool.free == 0
    with pytest.raises(RuntimeError, match="out of pages"):
        s.step()                            # slot 2 needs a fifth page
    with pytest.raises(RuntimeError, match="out of pages"):
        s.prefill([b], slots=[0])           # (nothing to give back)
    s.release([3])                          # of its pages one comes free
    assert s.pool.free == 1
    s.release([2])
    step(28)
    assert s.pool.used == 7                 # 51 tokens
    got = np.stack(got)
    assert np.abs(got - want).max() < 1e-4 * np.abs(want).max()
    assert (got.argmax(-1) == want.argmax(-1)).all()


def test_rope_scaling_reaches_past_the_models_window():
    """A context longer than max_position_embeddings with scaled positions:
    the same as a model whose tables are those."""
    from triton_llm.kernels import scaled_cos_sin
    scaling = {"type": "linear", "factor": 4.0}
    m, w = model()
    p = prompts_of(inputs.SMOL_TINY, [600])[0]
    with pytest.raises(ValueError, match="max_position_embeddings"):
        m.generate_paged([p], max_new_tokens=8)
    got = m.generate_paged([p], max_new_tokens=8, rope_scaling=scaling)[0]
    from smollm2_triton import SmolLM2Config
    kw = inputs.SMOL_TINY.config_kwargs()
    kw["max_position_embeddings"] = 700
    o = omodels.SmolLM2Oracle(SmolLM2Config(**kw), w)
    o.cos, o.sin = scaled_cos_sin(700, o.d, kw["rope_theta"], scaling)
    want, _ = o.generate(p, 8)
    assert got.tolist() == want[0].tolist()


# -- beam search ------------------------------------------------------------
def plain_beams(oracle, prompt, W, T, eos):
    """Beam search with one forward pass of the oracle per beam and step."""
    def logp(tokens):
        oracle.init_cache(len(tokens))
        x = oracle.forward_cached(np.array(tokens))[0, -1].astype(np.float64)
        return x - x.max() - np.log(np.exp(x - x.max()).sum())
    beams = [(0.0, [], False)]
    for _ in range(T):
        cand = []
        for b, (score, toks, done) in enumerate(beams):
            if done:
                cand.append((score, b, eos, toks, True))
                continue
            lp = logp(list(prompt) + toks)
            for t in np.argsort(-lp, kind="stable")[:W]:
                cand.append((score + lp[t], b, int(t), toks + [int(t)], int(t) == eos))
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        beams = [(c[0], c[3], c[4]) for c in cand[:W]]
    return beams


@pytest.mark.parametrize("W,T,P,graph", [(1, 6, 4, True), (3, 9, 4, True), (4, 12, 16, False),
                                         (4, 10, 5, True)])
def test_beam_search_against_plain_search(W, T, P, graph):
    """Weights five times larger than the parity tests': continuations whose
    scores differ by far more than rounding."""
    from smollm2_triton.paged import beam_search
    shape = inputs.SMOL_TINY
    m, w = model(weights=inputs.llama_weights_legacy(shape, 7, scale=0.1))
    m._init_gpu_weights()
    from smollm2_triton import SmolLM2Config
    o = omodels.SmolLM2Oracle(SmolLM2Config(**shape.config_kwargs()), w)
    prompts = prompts_of(shape, [5, 11, 8], seed=W)
    for eos in (None, int(plain_beams(o, prompts[0], W, T, -1)[0][1][T // 2])):
        got = beam_search(m.dev, prompts, W, T, eos, use_graph=graph, page_size=P)
        for p, beams in zip(prompts, got):
            want = plain_beams(o, p, W, T, -1 if eos is None else eos)
            assert [b[0].tolist() for b in beams] == [b[1] for b in want]
            assert np.abs([b[1] - x[0] for b, x in zip(beams, want)]).max() < 1e-3


def test_generate_beam():
    m, _ = model(dtype="bfloat16")
    p = prompts_of(inputs.SMOL_TINY, [6])
    one = m.generate_beam(p, beams=1, max_new_tokens=10)[0]
    want = m.generate_batch(p, max_new_tokens=10)[0][6:]
    assert one[0][0].tolist() == want.tolist()
    many = m.generate_beam(p, beams=5, max_new_tokens=10, length_penalty=1.0)[0]
    assert len(many) == 5 and many[0][1] >= many[-1][1]
    assert len({tuple(b[0].tolist()) for b in many}) == 5
    with pytest.raises(ValueError, match="beams"):
        m.generate_beam(p, beams=33)
    with pytest.raises(ValueError, match="window"):
        m.generate_beam(p, beams=2, window=8)
    with pytest.raises(ValueError, match="max_position_embeddings"):
        m.generate_beam(p, beams=2, max_new_tokens=600)
