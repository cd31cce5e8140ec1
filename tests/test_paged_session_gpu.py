"""What a PagedSession holds on the GPU and on the host besides its pages, and the
states that it refuses (on a B200)."""

from __future__ import annotations

import numpy as np
import pytest

import inputs

pytestmark = pytest.mark.gpu

SHAPE = inputs.SMOL_TINY


@pytest.fixture(scope="module")
def weights():
    from smollm2_triton import SmolLM2Config, SmolLM2ForCausalLM
    m = SmolLM2ForCausalLM(SmolLM2Config(**SHAPE.config_kwargs()),
                           inputs.llama_weights_legacy(SHAPE, 42), dtype="bfloat16")
    m._init_gpu_weights()
    return m


@pytest.fixture(autouse=True)
def no_device_errors():
    from triton_llm import gpu
    gpu.device_error(reset=True)
    yield
    assert gpu.device_error(reset=True) == 0


def prompt(n, seed=0):
    return np.random.default_rng(seed).integers(0, SHAPE.vocab_size, n).astype(np.int32)


def test_windowed_prefill_keeps_its_scratch_to_itself(weights):
    """The rows of a windowed prompt take a workspace that goes with the session,
    none of those that the library stream keeps for good."""
    from smollm2_triton.paged import PagedSession
    from triton_llm.kernels import paged
    before = set(paged._workspaces)
    s = PagedSession(weights.dev, 2, 300, page_size=16, window=40, sinks=2)
    for n in (70, 290, 20):
        s.prefill([prompt(n)], slots=[1])
    assert set(paged._workspaces) == before


def test_prompts_stage_their_own_rows(weights, monkeypatch):
    """A prompt admitted into a session of many slots stages its own keys and
    values, not places for every slot; results are the contiguous session's."""
    from smollm2_triton.engine import LlamaSession
    from smollm2_triton.paged import PagedSession
    from triton_llm import gpu
    prompts, slots = [prompt(33, 1), prompt(70, 2)], [9, 3]
    want = LlamaSession(weights.dev, 12, 100).prefill(prompts, slots=slots)
    for kw in (dict(), dict(window=80)):
        s = PagedSession(weights.dev, 12, 100, page_size=16, **kw)
        taken, allocate = [], gpu.allocate
        monkeypatch.setattr(gpu, "allocate", lambda shape, *a: taken.append(shape)
                            or allocate(shape, *a))
        got = s.prefill(prompts, slots=slots)
        monkeypatch.undo()
        staged = [x for x in taken if len(x) == 4]
        assert staged and all(x[0] == 2 for x in staged)
        assert np.abs(got - want).max() < 1e-4 * np.abs(want).max()
        # and the pages hold them: the next tokens agree too
        c = LlamaSession(weights.dev, 12, 100)
        c.prefill(prompts, slots=slots)
        for _ in range(4):
            s.step()
            c.step()
            a, b = s.logits.to_numpy()[slots], c.logits.to_numpy()[slots]
            assert np.abs(a - b).max() < 1e-4 * np.abs(b).max()


def test_idle_slots_of_a_session_shorter_than_a_page(weights):
    """An idle slot stays below max_seq (and the rotary tables' last position)
    however long the others go on."""
    from smollm2_triton.paged import PagedSession
    s = PagedSession(weights.dev, 2, 20, page_size=64,
                     rope_scaling={"type": "linear", "factor": 2.0})
    for seed in range(4):
        s.prefill([prompt(10, seed)], slots=[1])
        for _ in range(10):
            s.step()
            assert s._pos[0] <= 20 and s.pos.to_numpy()[0] <= 20


def test_set_state_refusals_change_nothing(weights):
    from smollm2_triton.paged import PagedSession
    s = PagedSession(weights.dev, 3, 100, page_size=16)
    p = prompt(40)
    s.prefill([p], slots=[1])
    alone = PagedSession(weights.dev, 3, 100, page_size=16)
    alone.prefill([p], slots=[1])
    for pos, ids in [([1, 101, 3], [0, 0, 0]), ([1, 2], [0, 0]), ([1, 2, 3, 4], [0] * 4),
                     ([1, -2, 3], [0, 0, 0]), ([1, 2, 3], [0, 0])]:
        with pytest.raises(ValueError, match="set_state"):
            s.set_state(np.array(pos), np.array(ids))
        assert s.pool.used == 3
    for _ in range(10):
        s.step()
        alone.step()
        assert (s.logits.to_numpy()[1] == alone.logits.to_numpy()[1]).all()
    s.set_state(np.array([100, 0, 16]), np.zeros(3, np.int32))
    assert s.pool.used == 7 + 1 + 1


def test_generate_paged_holds_what_its_sequences_need(weights, monkeypatch):
    """One long prompt among short ones does not make every sequence's pages as
    many as its own."""
    from smollm2_triton import paged
    made, init = [], paged.PagedSession._cache_buffers

    def record(self):
        made.append(self.n_pages)
        init(self)
    monkeypatch.setattr(paged.PagedSession, "_cache_buffers", record)
    prompts = [prompt(n, n) for n in (90, 3, 16, 1)]
    got = weights.generate_paged(prompts, max_new_tokens=17, page_size=16)
    assert made == [7 + 2 + 3 + 2]           # of 107, 20, 33 and 18 tokens
    want = weights.generate_batch(prompts, max_new_tokens=17)
    assert [g.tolist() for g in got] == [w.tolist() for w in want]
    weights.generate_paged(prompts, max_new_tokens=17, page_size=16, n_pages=20)
    assert made[-1] == 20
