"""RoPE (drop-in for triton_llm/kernels/rope.py).

``precompute_cos_sin`` builds the fp32 tables on the host exactly as the
reference does (rope.py:110-121: float32 positions and pair indices, numpy
cos/sin of their outer product); ``apply_rope`` rotates rows in place on the
GPU. In the decode step the rotation is fused into the QKV projection
epilogue (see kernels.linear), which writes K straight into the cache.
"""

from __future__ import annotations

import numpy as np

from triton_llm import gpu, _lib


def precompute_cos_sin(max_seq_len: int, d_k: int, theta: float = 100000.0):
    """Tables (max_seq_len, d_k // 2) float32: cos/sin(p * theta^(-2i/d_k))."""
    if max_seq_len < 1:
        raise ValueError(f"max_seq_len must be >= 1, got {max_seq_len}")
    if d_k < 2 or d_k % 2 != 0:
        raise ValueError(f"d_k must be even and >= 2, got {d_k}")
    if theta <= 0:
        raise ValueError(f"theta must be > 0, got {theta}")
    half = d_k // 2
    positions = np.arange(max_seq_len, dtype=np.float32)
    indices = np.arange(half, dtype=np.float32)
    freqs = 1.0 / (theta ** (2 * indices / d_k))
    angles = np.outer(positions, freqs)
    return np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)


def precompute_cos_sin_device(max_seq_len: int, d_k: int, theta: float = 100000.0):
    c, s = precompute_cos_sin(max_seq_len, d_k, theta)
    return gpu.to_device(c), gpu.to_device(s)


def scaled_cos_sin(max_seq_len: int, d_k: int, theta: float = 100000.0, scaling=None):
    """Tables (max_seq_len, d_k // 2) float32 for contexts longer than a model
    was trained on (no counterpart in the reference, whose window stays at the
    trained one). Pair i turns by ``position * f_i``, f_i = theta^(-2i/d_k)
    changed by ``scaling``, a dict with ``type`` (or ``rope_type``) and ``factor``:

    * ``None`` or ``"default"``: unchanged;
    * ``"linear"``: f_i / factor;
    * ``"ntk"``: theta * factor^(d_k / (d_k - 2)) in place of theta, so that the
      fastest pair stays and the slowest is divided by factor;
    * ``"llama3"``: by the pair's turns within
      ``original_max_position_embeddings`` tokens: pairs of more than
      ``high_freq_factor`` turns stay, those of fewer than ``low_freq_factor``
      are divided by factor, a ramp in 1 / wavelength between;
    * ``"yarn"``: a ramp over the pair index between the pairs that make
      ``beta_fast`` (32) and ``beta_slow`` (1) turns in the original context,
      and cos and sin times ``attention_factor`` (0.1 ln(factor) + 1).

    Angles are formed in 64 bits: at position 10^5 an fp32 product is off by up
    to 0.004 radians.
    """
    if max_seq_len < 1:
        raise ValueError(f"max_seq_len must be >= 1, got {max_seq_len}")
    if d_k < 2 or d_k % 2 != 0:
        raise ValueError(f"d_k must be even and >= 2, got {d_k}")
    if theta <= 0:
        raise ValueError(f"theta must be > 0, got {theta}")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    i = np.arange(d_k // 2, dtype=np.float64)
    freq = theta ** (-2 * i / d_k)
    size = 1.0
    if kind != "default":
        factor = float(scaling.get("factor", 0))
        if not factor >= 1:
            raise ValueError(f"rope scaling factor must be >= 1, got {scaling.get('factor')}")
    if kind in ("llama3", "yarn"):
        orig = scaling.get("original_max_position_embeddings")
        if not orig or orig <= 0:
            raise ValueError(f"{kind} rope scaling needs original_max_position_embeddings")
        turns = orig * freq / (2 * np.pi)
    if kind == "linear":
        freq = freq / factor
    elif kind == "ntk":
        if d_k < 4:
            raise ValueError("ntk rope scaling needs d_k >= 4")
        freq = (theta * factor ** (d_k / (d_k - 2))) ** (-2 * i / d_k)
    elif kind == "llama3":
        low, high = scaling.get("low_freq_factor", 1.0), scaling.get("high_freq_factor", 4.0)
        if not 0 < low < high:
            raise ValueError(f"low_freq_factor ({low}) must be in (0, high_freq_factor={high})")
        keep = np.clip((turns - low) / (high - low), 0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    elif kind == "yarn":
        fast, slow = scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0)
        if not 0 < slow < fast:
            raise ValueError(f"beta_slow ({slow}) must be in (0, beta_fast={fast})")

        def pair(n):   # the (real) index of the pair that makes n turns
            return d_k * np.log(orig / (n * 2 * np.pi)) / (2 * np.log(theta))
        first = max(np.floor(pair(fast)), 0)
        last = min(np.ceil(pair(slow)), d_k - 1)
        keep = 1 - np.clip((i - first) / max(last - first, 0.001), 0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        size = float(scaling.get("attention_factor") or
                     (0.1 * np.log(factor) + 1 if factor > 1 else 1.0))
    elif kind != "default":
        raise ValueError(f"unknown rope scaling {kind!r}")
    angle = np.arange(max_seq_len, dtype=np.float64)[:, None] * freq
    return ((np.cos(angle) * size).astype(np.float32),
            (np.sin(angle) * size).astype(np.float32))


def apply_rope(x_dev: "gpu.DeviceTensor", cos_dev: "gpu.DeviceTensor",
               sin_dev: "gpu.DeviceTensor", seq_len: int,
               position_offset: int = 0) -> "gpu.DeviceTensor":
    """In-place RoPE of x (n_rows, d_k); row r at (r % seq_len) + offset."""
    n_rows, d_k = x_dev.shape
    if d_k < 2 or d_k % 2 != 0:
        raise ValueError(f"d_k must be even and >= 2, got {d_k}")
    half = d_k // 2
    if len(cos_dev.shape) != 2 or len(sin_dev.shape) != 2:
        raise ValueError("cos_dev and sin_dev must be 2D tensors")
    if tuple(cos_dev.shape) != tuple(sin_dev.shape):
        raise ValueError(f"cos_dev and sin_dev shape mismatch: {cos_dev.shape} vs {sin_dev.shape}")
    if cos_dev.shape[1] != half:
        raise ValueError(f"cos_dev last dim must be d_k // 2 ({half}), got {cos_dev.shape[1]}")
    if n_rows == 0:
        return x_dev
    if seq_len < 1:
        raise ValueError(f"seq_len must be >= 1, got {seq_len}")
    if position_offset < 0:
        raise ValueError(f"position_offset must be >= 0, got {position_offset}")
    if position_offset + seq_len > cos_dev.shape[0]:
        raise ValueError(
            f"position_offset ({position_offset}) + seq_len ({seq_len}) "
            f"exceeds cos/sin table size ({cos_dev.shape[0]})")
    if n_rows % seq_len != 0:
        raise ValueError(f"Total rows ({n_rows}) must be a multiple of seq_len ({seq_len})")
    _lib.call("tllm_rope", x_dev.ptr, cos_dev.ptr, sin_dev.ptr, n_rows, d_k,
              int(seq_len), int(position_offset), None)
    return x_dev
