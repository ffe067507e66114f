"""Position rotation of a step's queries and keys, appended to a paged KV cache on the way (HIP kernel).

The reference rotates in its model code and stores then (prism_infer/layers/
rotary_embedding.py, prism_infer/ops/kv_cache_store.py); here one launch reads q, k
and v once, writes the rotated queries, and stores the rotated keys and the values.

- q: [tokens, num_heads, head_dim], key and value: [tokens, kv_heads, head_dim], one
  dtype of bf16, fp16 and fp32, head dims contiguous, any other strides (views of a
  packed projection are read in place);
- cos_sin: fp32 [max_positions, rotary_dim], the cosines of a position's
  ``rotary_dim / 2`` angles and then their sines; the first rotary_dim dims of a head
  are rotated, dims ``i`` and ``i + rotary_dim / 2`` as a pair, or ``2 i`` and
  ``2 i + 1`` with ``interleaved``, and the others stay;
- positions: int32 [tokens], or [axes, tokens] with ``position_axes``, int32
  [rotary_dim / 2], the row that each angle goes by (text, height and width of
  multimodal positions, in sections or alternating).  A pair whose position is
  outside the table, or whose axis is none of the rows, becomes NaN;
- the caches, scales and slots are those of ``store_kvcache``.  What is stored is bit
  for bit what ``store_kvcache`` stores of the rotated keys, which are rounded to
  their dtype first.  Tokens with slots that are negative or behind the cache are
  rotated and not stored.  Slots are distinct: one that several tokens name holds
  parts of any of them.

There is no backward pass: inputs that require gradients are refused while gradients
are recorded.
"""

from __future__ import annotations

import torch

from prism_infer import _native, observability
from prism_infer.observability import profile_region
from prism_infer.ops.kv_cache_store import _store_profile_region, _validate_store_inputs

HAS_HIP_KERNELS = _native.available()
_HOST = _native.host_ops()

ROTARY_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _validate_rotation(q, key, cos_sin, positions, position_axes) -> None:
    if q.ndim != 3 or q.shape[0] != key.shape[0] or q.shape[2] != key.shape[2]:
        raise ValueError(f"q must be [tokens={key.shape[0]}, num_heads, head_dim={key.shape[2]}], got {list(q.shape)}")
    if cos_sin.ndim != 2 or cos_sin.shape[1] % 2 or not 0 < cos_sin.shape[1] <= q.shape[2]:
        raise ValueError("cos_sin must be [max_positions, rotary_dim] with an even rotary_dim of at most "
                         f"head_dim={q.shape[2]}, got {list(cos_sin.shape)}")
    if cos_sin.dtype != torch.float32:
        raise ValueError(f"cos_sin must use torch.float32, got {cos_sin.dtype}")
    if positions.dtype != torch.int32:
        raise ValueError(f"positions must use torch.int32, got {positions.dtype}")
    if position_axes is None:
        if positions.ndim != 1 or positions.shape[0] != q.shape[0]:
            raise ValueError(f"positions must be [tokens={q.shape[0]}] without position_axes, got {list(positions.shape)}")
        return
    if positions.ndim != 2 or positions.shape[0] < 1 or positions.shape[1] != q.shape[0]:
        raise ValueError(f"positions must be [axes, tokens={q.shape[0]}] with position_axes, got {list(positions.shape)}")
    if position_axes.ndim != 1 or position_axes.numel() != cos_sin.shape[1] // 2 or position_axes.dtype != torch.int32:
        raise ValueError(f"position_axes must be torch.int32 [rotary_dim / 2 = {cos_sin.shape[1] // 2}], "
                         f"got {position_axes.dtype} {list(position_axes.shape)}")


def rotate_store_kvcache(
    q: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cos_sin: torch.Tensor,
    positions: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_scale_cache: torch.Tensor | None = None,
    v_scale_cache: torch.Tensor | None = None,
    *,
    position_axes: torch.Tensor | None = None,
    interleaved: bool = False,
    return_key: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Rotate q and key by their positions, store key and value; returns the rotated q (and key, with ``return_key``)."""

    # calls that the native checks accept; the rest, and every call while a
    # profiling provider is installed, goes on below
    if _HOST is not None and observability._region_provider is None:
        out = _HOST.rotate_store(q, key, value, cos_sin, positions, k_cache, v_cache, slot_mapping, k_scale_cache,
                                 v_scale_cache, position_axes, interleaved, return_key)
        if out is not None:
            return out
    scaled = _validate_store_inputs(key, value, k_cache, v_cache, slot_mapping, k_scale_cache, v_scale_cache)
    _validate_rotation(q, key, cos_sin, positions, position_axes)
    if q.dtype not in ROTARY_DTYPES or key.dtype != q.dtype or value.dtype != q.dtype:
        raise ValueError("q, key and value must have one dtype of float32/bfloat16/float16, "
                         f"got {q.dtype}, {key.dtype} and {value.dtype}")
    _native.lib()  # raises with the reason the library is unavailable
    caches = [k_cache, v_cache] + ([k_scale_cache, v_scale_cache] if scaled else [])
    tensors = [q, key, value, cos_sin, positions, slot_mapping, *caches] + ([] if position_axes is None else [position_axes])
    if not all(t.is_cuda for t in tensors) or any(t.device != q.device for t in tensors):
        raise RuntimeError("rotate_store_kvcache runs on the GPU: its tensors must share one CUDA device")
    if slot_mapping.dtype != torch.int32:
        raise ValueError("rotate_store_kvcache requires torch.int32 slot_mapping")
    if any(t.stride(-1) != 1 for t in (q, key, value)):
        raise RuntimeError("rotate_store_kvcache requires contiguous head dims")
    if not all(t.is_contiguous() for t in caches):
        raise RuntimeError("rotate_store_kvcache requires contiguous KV and scale caches")
    if torch.is_grad_enabled() and (q.requires_grad or key.requires_grad or value.requires_grad or cos_sin.requires_grad):
        raise RuntimeError("rotate_store_kvcache has no backward pass: call it without recording gradients")

    device = q.device
    lib = _native.device_lib(device)
    tokens, heads, dim = key.shape
    with torch.cuda.device(device):
        cos_sin, slot_mapping = cos_sin.contiguous(), slot_mapping.contiguous()
        positions = positions.contiguous()
        position_axes = None if position_axes is None else position_axes.contiguous()
        q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
        key_out = torch.empty(key.shape, dtype=q.dtype, device=device) if return_key else None
        if tokens > 0:
            with profile_region(
                _store_profile_region(scaled, k_cache), metadata={"cache_dtype": str(k_cache.dtype), "tokens": tokens},
            ):
                rc = lib.prism_kv_rotate_store(
                    q.data_ptr(), _native.row_strides(q), key.data_ptr(), _native.row_strides(key), value.data_ptr(),
                    _native.row_strides(value), _native.dtype_code(q.dtype), cos_sin.data_ptr(), cos_sin.shape[0],
                    cos_sin.shape[1], int(bool(interleaved)), positions.data_ptr(), tokens,
                    1 if position_axes is None else positions.shape[0],
                    None if position_axes is None else position_axes.data_ptr(), q_out.data_ptr(),
                    None if key_out is None else key_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                    _native.dtype_code(k_cache.dtype), k_scale_cache.data_ptr() if scaled else None,
                    v_scale_cache.data_ptr() if scaled else None, slot_mapping.data_ptr(), tokens, q.shape[1], heads, dim,
                    k_cache.numel() // (k_cache.shape[-2] * k_cache.shape[-1]) if k_cache.numel() else 0,
                    _native.stream_handle(device),
                )
                _native.check(rc, "rotate_store_kvcache")
    return q_out if key_out is None else (q_out, key_out)


__all__ = ["HAS_HIP_KERNELS", "rotate_store_kvcache"]
