"""Shared helpers of the kernel wrappers."""

from __future__ import annotations

import numpy as np

from triton_llm import _lib, gpu


def require_f32(t, name):
    if getattr(t, "is_bf16", False) or t.dtype != np.float32:
        raise ValueError(f"{name} must be float32, got "
                         f"{'bfloat16' if getattr(t, 'is_bf16', False) else t.dtype}")


def upload_f32(arr):
    return gpu.to_device(np.require(arr, dtype=np.float32, requirements=["C_CONTIGUOUS"]))


# dtype object -> TLLM code; numpy's and those of any array library whose
# tensors have data_ptr(), shape and dtype, met by the name of the dtype
_CODES = {np.dtype(np.float32): _lib.F32, np.dtype(np.int32): _lib.I32}
_NAMES = {"float32": _lib.F32, "bfloat16": _lib.BF16, "int32": _lib.I32}
_WORDS = {_lib.F32: "float32", _lib.BF16: "bfloat16", _lib.I32: "int32"}
_Device = gpu.DeviceTensor


def dtype_code(t, name="tensor"):
    """TLLM_F32, TLLM_BF16 or TLLM_I32 of a device tensor: a DeviceTensor, or
    an object with data_ptr(), shape and dtype (a torch CUDA tensor)."""
    if type(t) is _Device and t.is_bf16:
        return _lib.BF16
    code = _CODES.get(t.dtype)
    if code is None:
        code = _NAMES.get(str(t.dtype).rsplit(".", 1)[-1])
        if code is None:
            raise ValueError(f"{name} must be float32, bfloat16 or int32, got {t.dtype}")
        _CODES[t.dtype] = code
    return code


def strides(t):
    """Element strides of a device tensor (a DeviceTensor is contiguous)."""
    if type(t) is not _Device:
        try:
            return t.stride()
        except AttributeError:
            pass
    out, n = [], 1
    for s in reversed(t.shape):
        out.append(n)
        n *= int(s)
    return tuple(reversed(out))


def require_gpu(t, name):
    if type(t) is not _Device and not getattr(t, "is_cuda", True):
        raise ValueError(f"{name} is not on the GPU")


def on_device(t, name, code=None, shape=None):
    """Address of a contiguous device tensor, its type and shape checked."""
    if type(t) is not _Device:
        try:
            if ((code is None or _CODES[t.dtype] == code)
                    and (shape is None or t.shape == shape) and t.is_cuda
                    and t.is_contiguous()):
                return t.data_ptr()
        except (AttributeError, KeyError):
            pass
    if code is not None and dtype_code(t, name) != code:
        raise ValueError(f"{name} has dtype {'bfloat16' if getattr(t, 'is_bf16', 0) else t.dtype}"
                         f", expected {_WORDS[code]}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    require_gpu(t, name)
    if type(t) is not _Device:
        contiguous = getattr(t, "is_contiguous", None)
        if contiguous is not None and not contiguous():
            raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def device_of(t):
    """GPU index of a device tensor (a DeviceTensor is on the current one)."""
    index = None if type(t) is _Device else getattr(t, "get_device", None)
    return gpu.current_device() if index is None else index()
