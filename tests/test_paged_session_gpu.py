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
