"""Attention over 4-bit paged KV caches: what ``paged_decode_attention`` and ``paged_prefill_attention`` call for them.

No counterpart in the reference.  The payloads are ``torch.float4_e2m1fn_x2``
[blocks, page, kv_heads, head_dim / 2] and the exponents ``torch.float8_e8m0fnu``
[blocks, page, kv_heads, head_dim / 32], as ``store_kvcache`` fills them.  Queries are
bf16 or fp16, head_dim 64 or 128, any GQA group, pages of a multiple of 16 tokens.
Scores are exact products of queries and stored keys, summed in fp32.  Softmax
weights are rounded to the queries' type against fp32 sums (in decode after the values'
exponents are multiplied in, and for fp16 queries to 16 bits).
"""

from __future__ import annotations

import torch

from prism_infer import _native
from prism_infer.engine.kv_quantization import FP4_DTYPE
from prism_infer.ops.kv_cache_store import validate_fp4_scales

FP4_HEAD_DIMS = (64, 128)
FP4_PAGE_MULTIPLE = 16


def is_fp4(cache: torch.Tensor) -> bool:
    return cache.dtype == FP4_DTYPE


def validate_fp4_call(what: str, q, k_cache, v_cache, k_scale_cache, v_scale_cache, block_tables) -> None:
    """What both ops ask of a call over a 4-bit cache; its types and shapes first, then where the tensors live."""

    if q.ndim != 3:
        raise ValueError(f"q must be [tokens, num_heads, head_dim], got {list(q.shape)}")
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError("4-bit k_cache/v_cache must both be [num_blocks, block_size, num_kv_heads, head_dim / 2], "
                         f"got {k_cache.dtype} {list(k_cache.shape)} and {v_cache.dtype} {list(v_cache.shape)}")
    page_size, num_kv_heads, row = k_cache.shape[1:]
    if 2 * row != q.shape[2]:
        raise ValueError(f"head_dim mismatch: q={q.shape[2]}, cache={2 * row}")
    if num_kv_heads <= 0 or q.shape[1] <= 0 or q.shape[1] % num_kv_heads:
        raise ValueError(f"num_heads must be divisible by num_kv_heads, got {q.shape[1]} and {num_kv_heads}")
    validate_fp4_scales(k_cache, k_scale_cache, v_scale_cache)
    if block_tables.ndim != 2:
        raise ValueError(f"block_tables must be two-dimensional, got {list(block_tables.shape)}")
    if page_size <= 0 or page_size % FP4_PAGE_MULTIPLE:
        raise RuntimeError(f"{what} over 4-bit caches takes pages of a multiple of {FP4_PAGE_MULTIPLE} tokens, got {page_size}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f"{what} over 4-bit caches takes bf16 or float16 queries, got {q.dtype}")
    if q.shape[2] not in FP4_HEAD_DIMS:
        raise RuntimeError(f"{what} over 4-bit caches covers head_dim 64 and 128, got {q.shape[2]}")
    if torch.is_grad_enabled() and q.requires_grad:
        raise RuntimeError(f"{what} has no backward pass over 4-bit caches: call it without recording gradients")


def validate_fp4_devices(what: str, *tensors) -> None:
    _native.lib()  # raises with the reason the library is unavailable
    if not all(t.is_cuda for t in tensors) or any(t.device != tensors[0].device for t in tensors):
        raise RuntimeError(f"{what} requires all tensors on one GPU (there is no CPU fallback)")


def _aligned_scales(scales: torch.Tensor) -> torch.Tensor:
    """The exponents, or a copy where a row of them does not start on its own length."""

    row = scales.shape[-1]
    if (scales.stride(-1) == 1 and scales.data_ptr() % row == 0
            and all(n == 1 or s % row == 0 for n, s in zip(scales.shape[:-1], scales.stride()))):
        return scales
    return scales.clone(memory_format=torch.contiguous_format)


def launch_fp4(what: str, q, k_cache, v_cache, k_scale_cache, v_scale_cache, block_tables, context_lens, scale, *,
               max_context_len=None, cu_seqlens_q=None, batch=None, status=None):
    """Enqueue the attention of checked tensors; returns the output, with q's rows."""

    device = q.device
    lib = _native.device_lib(device)
    total_q, num_heads, head_dim = q.shape
    num_blocks, page_size, num_kv_heads, _ = k_cache.shape
    batch = total_q if batch is None else batch
    with torch.cuda.device(device):
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
        if total_q == 0:
            return out
        q, k_cache, v_cache = (_native.aligned_rows(t) for t in (q, k_cache, v_cache))
        k_scale_cache, v_scale_cache = _aligned_scales(k_scale_cache), _aligned_scales(v_scale_cache)
        context_lens = context_lens.contiguous()
        width = block_tables.shape[1]
        need = lib.prism_paged_fp4_workspace_bytes(int(cu_seqlens_q is not None), batch, total_q, num_heads, num_kv_heads,
                                                   head_dim, page_size, width)
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=device)
        rc = lib.prism_paged_fp4(
            q.data_ptr(), _native.dtype_code(q.dtype), _native.row_strides(q), k_cache.data_ptr(), v_cache.data_ptr(),
            _native.row_strides(k_cache), _native.row_strides(v_cache), k_scale_cache.data_ptr(), v_scale_cache.data_ptr(),
            _native.row_strides(k_scale_cache), _native.row_strides(v_scale_cache), block_tables.data_ptr(),
            _native.strides(block_tables), context_lens.data_ptr(),
            None if max_context_len is None else max_context_len.data_ptr(),
            None if cu_seqlens_q is None else cu_seqlens_q.data_ptr(), out.data_ptr(), _native.strides(out), batch, total_q,
            num_heads, num_kv_heads, head_dim, page_size, num_blocks, width, float(scale),
            None if status is None else status.data_ptr(), None, workspace.data_ptr(), need, _native.stream_handle(device),
        )
    _native.check(rc, what)
    return out


__all__ = ["FP4_HEAD_DIMS", "is_fp4", "launch_fp4", "validate_fp4_call", "validate_fp4_devices"]
