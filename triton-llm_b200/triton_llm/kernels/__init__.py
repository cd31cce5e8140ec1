"""Kernel library (drop-in for triton_llm/kernels/__init__.py).

Every function launches hand-written sm_100a CUDA from libtllm.so; the
reference's names and signatures are kept, and the batched / fused entry
points used by the models are exported next to them.
"""

from .add import add
from .attention import attention
from .attention_gqa import attention_gqa, gqa_decode, DecodeWorkspace
from .attention_prefill import gqa_rows, gqa_prefill, prefill_blocks
from .beam import BeamWorkspace, beam_reorder, beam_select
from .embedding import embedding, embedding_dev
from .gelu import gelu
from .gemm import gemm
from .layernorm import layer_norm, layer_norm_dev
from .linear import Linear, LinearWorkspace, linear
from .paged import (PagedKV, PagedWorkspace, page_copy, paged_append, paged_attention,
                    paged_write)
from .rms_norm import rms_norm
from .rope import (apply_rope, precompute_cos_sin, precompute_cos_sin_device,
                   scaled_cos_sin)
from .softmax import softmax
from .swiglu import swiglu

__all__ = [
    "add",
    "attention",
    "attention_gqa",
    "embedding",
    "gelu",
    "gemm",
    "layer_norm",
    "rms_norm",
    "precompute_cos_sin",
    "apply_rope",
    "softmax",
    "swiglu",
    # batched / fused entry points of the B200 path
    "gqa_decode",
    "gqa_rows",
    "gqa_prefill",
    "prefill_blocks",
    "DecodeWorkspace",
    "embedding_dev",
    "layer_norm_dev",
    "precompute_cos_sin_device",
    "Linear",
    "LinearWorkspace",
    "linear",
    # paged cache and beam search
    "PagedKV",
    "PagedWorkspace",
    "paged_attention",
    "paged_append",
    "paged_write",
    "page_copy",
    "BeamWorkspace",
    "beam_select",
    "beam_reorder",
    "scaled_cos_sin",
]
