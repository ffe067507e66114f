"""Causal attention over packed prompts on MI355X (HIP kernel).

What the reference's attention layer takes from an external varlen attention
when nothing is cached in front of a prompt (prism_infer/layers/attention.py:
180-208): the prompts' own K/V, packed like their queries, no pages.

- q: [total_q, num_heads, head_dim], k and v: [total_k, num_kv_heads, head_dim],
  bf16 or fp16, head_dim 64 or 128, any strides (views of a packed projection
  are read in place; rows that do not start on 16 bytes are copied first);
- sequence i owns query rows ``cu_seqlens_q[i]:cu_seqlens_q[i + 1]`` and key rows
  ``cu_seqlens_k[i]:cu_seqlens_k[i + 1]``.  Its queries are its last tokens: query
  j of qlen sits at position ``klen - qlen + j`` and attends to keys 0 to there,
  so rows of a sequence with fewer keys than queries may see none;
- rows that see no key are zeros, and so are rows outside ``[cu_seqlens_q[0],
  cu_seqlens_q[-1])``, as a batch padded to a captured size has them.

The offsets stay on the device and the call does not synchronise: it can be
captured, and a replay follows the offsets of its time.  A sequence whose offsets
are out of order or outside the tensors is left out; its rows are unspecified, and
so are all rows where sequences share some.  A call takes up to 2**29 keys, and of
query rows (tokens times heads per kv head) up to 2**29 per kv head and fewer than
2**24 workgroups: a kv head has one per 128 rows, one per sequence and one more.
There is no backward pass: inputs that require gradients are refused while
gradients are recorded.
"""

from __future__ import annotations

import torch

from prism_infer import _native

HAS_HIP_KERNELS = _native.available()
_HOST = _native.host_ops()

PROMPT_HEAD_DIMS = (64, 128)
MAX_PROMPT_TOKENS = 2**29
PROMPT_DTYPES = (torch.bfloat16, torch.float16)


def _validate_prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, num_heads: int, num_kv_heads: int) -> None:
    same_tokens = cu_seqlens_k is None
    cu_seqlens_k = cu_seqlens_q if same_tokens else cu_seqlens_k
    if num_kv_heads <= 0 or num_heads <= 0 or num_heads % num_kv_heads:
        raise ValueError(
            "num_heads must be divisible by num_kv_heads, "
            f"got num_heads={num_heads}, num_kv_heads={num_kv_heads}"
        )
    if q.ndim != 3 or q.shape[1] != num_heads:
        raise ValueError(f"q must be [tokens, num_heads={num_heads}, head_dim], got {list(q.shape)}")
    if k.ndim != 3 or k.shape != v.shape or k.shape[1] != num_kv_heads or k.shape[2] != q.shape[2]:
        raise ValueError(
            f"k and v must be [tokens, num_kv_heads={num_kv_heads}, head_dim={q.shape[2]}], "
            f"got {list(k.shape)} and {list(v.shape)}"
        )
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError(f"q, k and v dtype mismatch: {q.dtype}, {k.dtype}, {v.dtype}")
    for name, cu in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        if cu.ndim != 1 or cu.numel() < 1 or cu.dtype != torch.int32:
            raise ValueError(f"{name} must be a one-dimensional torch.int32 tensor of batch + 1 offsets, "
                             f"got {cu.dtype} {list(cu.shape)}")
    if cu_seqlens_k.numel() != cu_seqlens_q.numel():
        raise ValueError("cu_seqlens_q and cu_seqlens_k must have the same length, "
                         f"got {cu_seqlens_q.numel()} and {cu_seqlens_k.numel()}")
    if same_tokens and k.shape[0] != q.shape[0]:
        raise ValueError("without cu_seqlens_k q, k and v must have the same tokens, "
                         f"got {q.shape[0]} and {k.shape[0]}")


def prompt_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    *,
    num_heads: int,
    num_kv_heads: int,
    scale: float,
    cu_seqlens_k: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attend each packed prompt to its own keys, causally; returns [total_q, num_heads, head_dim]."""

    # calls that the native checks accept; the rest goes on below
    if _HOST is not None:
        out = _HOST.prompt(q, k, v, cu_seqlens_q, cu_seqlens_k, num_heads, num_kv_heads, scale)
        if out is not None:
            return out
    _validate_prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, num_heads, num_kv_heads)
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    if max(q.shape[0], k.shape[0]) > MAX_PROMPT_TOKENS:
        raise RuntimeError(f"prompt_attention takes at most {MAX_PROMPT_TOKENS} tokens, got {q.shape[0]} and {k.shape[0]}")
    _native.lib()  # raises with the reason the library is unavailable
    tensors = (q, k, v, cu_seqlens_q, cu_seqlens_k)
    if not all(t.is_cuda for t in tensors) or any(t.device != q.device for t in tensors):
        raise RuntimeError("prompt_attention runs on the GPU: q, k, v and the offsets must share one CUDA device")
    if q.dtype not in PROMPT_DTYPES:
        raise RuntimeError(f"the HIP prompt attention kernel takes bf16 or float16, got {q.dtype}")
    if q.shape[2] not in PROMPT_HEAD_DIMS:
        raise RuntimeError(f"the HIP prompt attention kernel covers head_dim 64 and 128, got {q.shape[2]}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        raise RuntimeError("prompt_attention has no backward pass: call it without recording gradients")

    lib = _native.device_lib(q.device)
    q, k, v = map(_native.aligned_rows, (q, k, v))
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    with torch.cuda.device(q.device):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        batch = cu_seqlens_q.numel() - 1
        # scratch for split keys (static shapes only; 0 bytes where none are split)
        ws_bytes = lib.prism_prompt_attention_workspace_bytes(batch, q.shape[0], k.shape[0], num_heads, num_kv_heads, q.shape[2])
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes > 0 else None
        rc = lib.prism_prompt_attention(
            q.data_ptr(), _native.row_strides(q), k.data_ptr(), _native.row_strides(k), v.data_ptr(), _native.row_strides(v),
            _native.dtype_code(q.dtype), cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
            out.data_ptr(), _native.strides(out), batch, q.shape[0], k.shape[0],
            num_heads, num_kv_heads, q.shape[2], float(scale),
            workspace.data_ptr() if workspace is not None else None, ws_bytes, _native.stream_handle(q.device),
        )
    _native.check(rc, "prompt_attention")
    return out


__all__ = ["HAS_HIP_KERNELS", "prompt_attention"]
