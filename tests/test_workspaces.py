"""Workspaces of the paged cache's and beam search's operators: when they may be
used and released, and how large they get (CPU: the device is a fake)."""

from __future__ import annotations

import ctypes

import pytest

from triton_llm import _lib, gpu
from triton_llm.kernels import BeamWorkspace, PagedWorkspace, beam_select


class FakeDevice:
    """Records the library's calls on memory and streams; the rest goes through."""

    NAMES = ("tllm_malloc", "tllm_free", "tllm_malloc_static", "tllm_free_static",
             "tllm_memset", "tllm_synchronize", "tllm_stream_synchronize",
             "tllm_device_synchronize", "tllm_get_device", "tllm_set_device",
             "tllm_beam_select")

    def __init__(self, real):
        self._real, self.log, self.refuse = real, [], None

    def __getattr__(self, name):
        if name not in self.NAMES:
            return getattr(self._real, name)

        def call(*args):
            self.log.append(name)
            if name == "tllm_beam_select":
                self.select = args[0]
            if name in ("tllm_malloc", "tllm_malloc_static"):
                args[0]._obj.value = 1 << 20
            return _lib.ERR_CUDA if name == self.refuse else 0
        return call


@pytest.fixture
def device(monkeypatch):
    fake = FakeDevice(_lib.load())
    monkeypatch.setattr(_lib, "_lib", fake)
    monkeypatch.setattr(gpu, "_initialized", True)
    return fake


@pytest.mark.parametrize("make", [lambda: PagedWorkspace(4, 24, 8, 128),
                                  lambda: BeamWorkspace(2, 4, 1000, 4)])
def test_ready_for_any_stream(device, make):
    """A workspace is zero-filled when its constructor returns, whatever stream
    uses it next; its memory is none of the library stream's pool, which would
    hand it out again while another stream's work still uses it."""
    ws = make()
    log = device.log
    fill = max(i for i, name in enumerate(log) if name == "tllm_memset")
    assert any(name in ("tllm_synchronize", "tllm_stream_synchronize") for name in log[fill:])
    assert "tllm_malloc_static" in log and "tllm_malloc" not in log
    n, at = log.count("tllm_malloc_static"), len(log)
    del ws
    assert log.count("tllm_free_static") == n and "tllm_free" not in log
    assert "tllm_device_synchronize" in log[at:log.index("tllm_free_static")]


def test_kept_where_the_device_cannot_be_waited_for(device):
    """Released in the middle of a graph capture, a workspace's memory stays: the
    work that uses it may not be over."""
    ws, free = PagedWorkspace(4, 24, 8, 128), len(device.log)
    device.refuse = "tllm_device_synchronize"
    del ws
    assert "tllm_device_synchronize" in device.log[free:]
    assert "tllm_free_static" not in device.log


def test_attention_scratch_is_bounded():
    """Calls of many rows (the prompt rows of a windowed prefill): their rows fill
    the GPU, so that splits are few or none; the scratch stays within 512 MB. A
    decode batch keeps its 8 splits and more."""
    lib = _lib.load()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()

    def need(rows, heads, kv, dim):
        assert lib.tllm_paged_attention_workspace(rows, heads, kv, dim, ctypes.byref(a),
                                                  ctypes.byref(b)) == _lib.OK
        return a.value
    for rows, heads, kv, dim in [(16384, 24, 8, 128), (32768, 32, 8, 128), (131072, 9, 3, 64),
                                 (1 << 20, 8, 1, 128)]:
        # (two parts of a share for each of 296 CTAs and 512 rows, if that is more)
        shares = rows // 512 * 296 * 2 * (heads // kv) * (dim + 2) * 4
        assert need(rows, heads, kv, dim) <= max(1 << 29, shares)
    for rows in (1, 64, 512):
        row = 24 * 2 * (128 + 2) * 4
        assert need(rows, 24, 8, 128) >= 8 * rows * row


class Tensor:
    """A described tensor, for calls that do not reach the device."""

    def __init__(self, shape, dtype="float32"):
        self.shape, self.dtype, self.is_cuda = tuple(shape), f"any.{dtype}", True

    def data_ptr(self):
        return 4096

    def is_contiguous(self):
        return True

    def get_device(self):
        return 0


def test_beam_scratch_of_ever_other_shapes(device, monkeypatch):
    """The library stream's own workspaces stay few whatever numbers of requests,
    beams, tokens and continuations come, and are large enough for each."""
    from triton_llm.kernels import paged
    kept = {}
    monkeypatch.setattr(paged, "_workspaces", kept)
    real, need = device._real, ctypes.c_size_t()
    for groups in (1, 3, 5, 16, 37, 100, 1000):
        for beams in (1, 2, 5, 8):
            for vocab in (100, 5000, 32000, 128256):
                for k in {1, 3, beams, 2 * beams, 64}:
                    assert real.tllm_beam_workspace(groups, beams, vocab, k,
                                                    ctypes.byref(need)) == _lib.OK
                    beam_select(Tensor((groups * beams, vocab)), Tensor((groups, beams)),
                                Tensor((groups, k)), Tensor((groups, k), "int32"),
                                Tensor((groups, k), "int32"))
                    used = packed(device.select)
                    assert used >= need.value
    assert len(kept) <= 14 * 7
    assert sum(ws.nbytes for ws in kept.values()) < 64 << 20


def packed(step):
    """workspace_bytes of a packed tllm_beam_step."""
    return _lib.BEAM_STEP.unpack(step)[8]


@pytest.mark.gpu
def test_dropped_while_another_stream_works():
    """A workspace made for one call on another stream and dropped at once, with
    the library stream writing over whatever memory it gets meanwhile."""
    import numpy as np
    from triton_llm.kernels import PagedKV, paged_attention
    rng = np.random.default_rng(0)
    R, K, P, n = 8, 8, 64, 256
    kv = PagedKV(*[gpu.to_device_bf16(rng.standard_normal((n, K, P, 128), np.float32))
                   for _ in range(2)],
                 gpu.to_device(rng.integers(0, n, (R, 100)).astype(np.int32)))
    q = gpu.to_device(rng.standard_normal((R, 24, 128), np.float32))
    lens = gpu.to_device(np.linspace(1, 6400, R).astype(np.int32))
    x = gpu.to_device(rng.standard_normal((64, 60000), np.float32))
    zero = gpu.zeros((8, 8))
    out = gpu.zeros((R, 24, 128))
    best = [gpu.zeros((8, 8), d) for d in (np.float32, np.int32, np.int32)]
    paged_attention(kv, q, lens, out)
    beam_select(x, zero, *best)
    want = [t.to_numpy() for t in [out, *best]]
    s = ctypes.c_void_p()
    _lib.call("tllm_stream_create", ctypes.byref(s))
    for _ in range(20):
        for t in [out, *best]:
            gpu.memset(t, 0)
        gpu.synchronize()
        paged_attention(kv, q, lens, out, stream=s, workspace=PagedWorkspace(R, 24, K, 128))
        beam_select(x, zero, *best, stream=s, workspace=BeamWorkspace(8, 8, 60000, 8))
        for _ in range(4):
            gpu.memset(gpu.allocate((1 << 22,), np.int32), 0xff)
        gpu.stream_synchronize(s)
        gpu.synchronize()
        for t, w in zip([out, *best], want):
            assert (t.to_numpy() == w).all()
    _lib.call("tllm_stream_destroy", s)
    assert gpu.device_error() == 0
