"""Rows of a paged KV cache read back as 16- or 32-bit rows (HIP kernel).

The inverse of :func:`store_kvcache`, with its cache layouts: 16- and 32-bit
caches, FP8 with and without token-head scales, 4-bit ones.  No counterpart in the
reference, whose caches are read by attention alone; here it hands stored tokens
to whatever takes plain rows (``prompt_attention``, a cache of another format).
"""

from __future__ import annotations

import torch

from prism_infer import _native
from prism_infer.ops.kv_cache_store import (
    SLOT_MAPPING_TENSOR_RANK,
    SUPPORTED_KV_CACHE_RANKS,
    _validate_scale_store_inputs,
    is_fp4_cache_tensor,
)

HAS_HIP_KERNELS = _native.available()
_HOST = _native.host_ops()

LOAD_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def load_kvcache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_scale_cache: torch.Tensor | None = None,
    v_scale_cache: torch.Tensor | None = None,
    *,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """(key, value), each [tokens, kv_heads, head_dim] of ``dtype``: what the slots hold.

    Payload times scale in fp32, rounded once to ``dtype``; zeros for slots that are
    negative or behind the cache.  head_dim is a multiple of 8.
    """

    # calls that the native checks accept; the rest goes on below
    if _HOST is not None and dtype in LOAD_DTYPES:
        out = _HOST.load(k_cache, v_cache, slot_mapping, k_scale_cache, v_scale_cache, _native.dtype_code(dtype))
        if out is not None:
            return out
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError("K/V payload caches must have matching shape and dtype")
    if k_cache.ndim not in SUPPORTED_KV_CACHE_RANKS:
        raise ValueError("K/V payload caches must be [slots, heads, dim] or [blocks, page, heads, dim]")
    if slot_mapping.ndim != SLOT_MAPPING_TENSOR_RANK:
        raise ValueError("slot_mapping must contain one flat slot per token")
    if dtype not in LOAD_DTYPES:
        raise ValueError(f"dtype must be one of float32/bfloat16/float16, got {dtype}")
    scaled = _validate_scale_store_inputs(k_cache, k_scale_cache, v_scale_cache)
    _native.lib()  # raises with the reason the library is unavailable
    tensors = [k_cache, v_cache, slot_mapping] + ([k_scale_cache, v_scale_cache] if scaled else [])
    if not all(t.is_cuda for t in tensors) or any(t.device != k_cache.device for t in tensors):
        raise RuntimeError("load_kvcache runs on the GPU: caches, scales and slots must share one CUDA device")
    if slot_mapping.dtype != torch.int32:
        raise ValueError("load_kvcache requires torch.int32 slot_mapping")
    if not all(t.is_contiguous() for t in tensors):
        raise RuntimeError("load_kvcache requires contiguous caches, scales and slots")
    device = k_cache.device
    heads, dim = k_cache.shape[-2:]
    slots = k_cache.numel() // (heads * dim) if k_cache.numel() else 0
    dim = 2 * dim if is_fp4_cache_tensor(k_cache) else dim
    tokens = slot_mapping.numel()
    lib = _native.device_lib(device)
    with torch.cuda.device(device):
        key, value = (torch.empty((tokens, heads, dim), dtype=dtype, device=device) for _ in range(2))
        if key.numel():
            rc = lib.prism_kv_load(
                k_cache.data_ptr(), v_cache.data_ptr(), _native.dtype_code(k_cache.dtype),
                k_scale_cache.data_ptr() if scaled else None, v_scale_cache.data_ptr() if scaled else None,
                slot_mapping.data_ptr(), key.data_ptr(), value.data_ptr(), _native.dtype_code(dtype), tokens, heads, dim,
                slots, _native.stream_handle(device),
            )
            _native.check(rc, "load_kvcache")
    return key, value


__all__ = ["HAS_HIP_KERNELS", "load_kvcache"]
