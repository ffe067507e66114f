"""A step's attention metadata, built on the GPU from the requests' lengths.

The reference prepares a step on the host, list by list
(prism_infer/engine/input_preparation.py:324 slot mapping, :571-603 packing), and
so does :func:`prism_infer.engine.decode_attention.pack_decode_metadata`.  Here
the lengths, the held blocks and the free blocks are on the device and stay
there: one launch makes the offsets, the context lengths, the block tables with
the blocks that the new tokens need, and every new token's position and slot.

A :class:`StepMetadata` has the attributes that the ops read: ``slot_mapping``
for ``store_kvcache``; ``cu_seqlens_q`` for ``prompt_attention``; it is a
``context`` of ``paged_prefill_attention`` and, for steps of one token per
request, the metadata of ``PagedKVDecodeAttention``.  The next step's held
blocks, cached lengths and ``free_start`` are this one's ``block_tables``,
``context_lens`` and ``next_free``, without a host copy in between.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from prism_infer import _native

_HOST = _native.host_ops()

MAX_STEP_REQUESTS = 8192
MAX_STEP_TOKENS = 2**30
_FITS = 2**31 - 1


@dataclass(slots=True)
class StepMetadata:
    packed: torch.Tensor           # int32, all of the below
    slot_mapping: torch.Tensor     # int32 [num_tokens], -1 behind the last token
    positions: torch.Tensor        # int32 [num_tokens], 0 behind the last token
    cu_seqlens_q: torch.Tensor     # int32 [B + 1]
    context_lens: torch.Tensor     # int32 [B], cached + new tokens
    max_context_len: torch.Tensor  # int32, 0-dim
    next_free: torch.Tensor        # int32, 0-dim, first free block that was not taken
    first_misfit: torch.Tensor     # int32, 0-dim, lowest request that does not fit, or 2**31 - 1
    block_tables: torch.Tensor     # int32 [B, W], -1 behind a request's last block

    @property
    def batch(self) -> int:
        return self.context_lens.numel()

    def check(self) -> "StepMetadata":
        """Raise if a request did not fit (waits for the step's launch)."""

        request = int(self.first_misfit)
        if request != _FITS:
            raise RuntimeError(
                f"step metadata: request {request} does not fit: a negative length, a context longer than its block "
                "table, more tokens than num_tokens, or too few free blocks"
            )
        return self


def _pad4(n: int) -> int:
    return -(-n // 4) * 4


def _views(packed: torch.Tensor, batch: int, width: int, num_tokens: int) -> StepMetadata:
    o = 2 * _pad4(num_tokens)
    ctx = o + batch + 1
    tail = ctx + batch
    tables = o + _pad4(2 * batch + 4)
    return StepMetadata(
        packed, packed[:num_tokens], packed[_pad4(num_tokens):_pad4(num_tokens) + num_tokens], packed[o:ctx],
        packed[ctx:tail], packed[tail], packed[tail + 1], packed[tail + 2],
        packed[tables:tables + batch * width].view(batch, width),
    )


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    if a.numel() == 0 or b.numel() == 0:
        return False

    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def build_step_metadata(
    block_tables: torch.Tensor,
    cached_lens: torch.Tensor,
    query_lens: torch.Tensor,
    *,
    block_size: int,
    num_tokens: int,
    free_blocks: torch.Tensor | None = None,
    free_start: torch.Tensor | None = None,
    out: StepMetadata | None = None,
) -> StepMetadata:
    """Build a step's metadata for ``query_lens`` new tokens behind ``cached_lens`` stored ones.

    ``block_tables`` [B, W] holds each request's blocks in its first
    ``ceil(cached / block_size)`` entries; the rest is ignored.  Blocks that new
    tokens need are taken from ``free_blocks``, request by request, from entry
    ``free_start`` (an int32 tensor of one value, default 0) on.  ``num_tokens``
    is the number of token rows, at most 2**30, which may exceed the tokens (padded
    rows get slot -1).  ``out`` is filled in place, as a captured graph's buffers are; it
    must not share memory with the inputs.  All tensors are int32 on one device.
    Nothing is synchronised: requests that do not fit get -1 where a block is
    missing, and :meth:`StepMetadata.check` reports them.  Held blocks are taken as
    they are: a token in one that is -1 gets slot -1, which ``check`` does not report.
    """

    # calls that the native checks accept; the rest goes on below
    if _HOST is not None and out is None:
        done = _HOST.step_metadata(block_tables, cached_lens, query_lens, block_size, num_tokens, free_blocks, free_start)
        if done is not None:
            return StepMetadata(*done)
    block_size, num_tokens = int(block_size), int(num_tokens)
    if block_size <= 0 or num_tokens < 0:
        raise ValueError(f"block_size must be positive and num_tokens not negative, got {block_size} and {num_tokens}")
    if block_size > _FITS or num_tokens > MAX_STEP_TOKENS:
        raise ValueError(f"block_size must be below 2**31 and num_tokens at most {MAX_STEP_TOKENS}, got {block_size} and {num_tokens}")
    if block_tables.ndim != 2 or cached_lens.ndim != 1 or query_lens.ndim != 1:
        raise ValueError("block_tables must be [B, W], cached_lens and query_lens [B], got "
                         f"{list(block_tables.shape)}, {list(cached_lens.shape)} and {list(query_lens.shape)}")
    batch, width = block_tables.shape
    if cached_lens.numel() != batch or query_lens.numel() != batch:
        raise ValueError("block_tables, cached_lens and query_lens must have one entry per request, got "
                         f"{batch}, {cached_lens.numel()} and {query_lens.numel()}")
    if free_blocks is not None and free_blocks.ndim != 1:
        raise ValueError(f"free_blocks must be one-dimensional, got {list(free_blocks.shape)}")
    if free_start is not None and free_start.numel() != 1:
        raise ValueError(f"free_start must hold one value, got {list(free_start.shape)}")
    inputs = [t for t in (block_tables, cached_lens, query_lens, free_blocks, free_start) if t is not None]
    if any(t.dtype != torch.int32 for t in inputs):
        raise ValueError(f"step metadata inputs must use torch.int32, got {[t.dtype for t in inputs]}")
    lib = _native.lib()  # raises with the reason the library is unavailable
    device = block_tables.device
    if any(not t.is_cuda or t.device != device for t in inputs):
        raise RuntimeError("build_step_metadata runs on the GPU: its inputs must share one CUDA device")
    if batch > MAX_STEP_REQUESTS:
        raise RuntimeError(f"build_step_metadata takes at most {MAX_STEP_REQUESTS} requests, got {batch}")
    lib = _native.device_lib(device)
    words = lib.prism_step_metadata_words(batch, width, num_tokens)
    if out is None:
        out = _views(torch.empty(words, dtype=torch.int32, device=device), batch, width, num_tokens)
    else:
        if (out.packed.device != device or out.packed.numel() != words or out.block_tables.shape != (batch, width)
                or out.slot_mapping.numel() != num_tokens):
            raise ValueError("out was made for other sizes or on another device")
        if any(_overlap(out.packed, t) for t in inputs):
            raise ValueError("out shares memory with the inputs")
    cached_lens, query_lens = cached_lens.contiguous(), query_lens.contiguous()
    free_blocks = None if free_blocks is None else free_blocks.contiguous()
    with torch.cuda.device(device):
        rc = lib.prism_step_metadata(
            block_tables.data_ptr(), _native.strides(block_tables), cached_lens.data_ptr(), query_lens.data_ptr(),
            None if free_blocks is None else free_blocks.data_ptr(), 0 if free_blocks is None else free_blocks.numel(),
            None if free_start is None else free_start.data_ptr(), batch, width, block_size, num_tokens,
            out.packed.data_ptr(), _native.stream_handle(device),
        )
    _native.check(rc, "build_step_metadata")
    return out


__all__ = ["MAX_STEP_REQUESTS", "StepMetadata", "build_step_metadata"]
