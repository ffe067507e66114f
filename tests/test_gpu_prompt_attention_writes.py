"""Prompt attention writes nothing but its output and its scratch, whatever the offsets, at every size of a batch."""

from __future__ import annotations

import pytest
import torch

from _attention16 import assert_within, attention64
from _helpers import require_gpu

pytestmark = pytest.mark.gpu

GUARD = 1 << 20  # bytes on either side of the output and of the scratch
MARK = 0xA5


def _guarded(nbytes):
    whole = torch.full((nbytes + 2 * GUARD,), MARK, dtype=torch.uint8, device="cuda")
    return whole, whole[GUARD:GUARD + nbytes]


def _call(q, k, v, cu):
    """The C entry with output and scratch inside marked buffers, whose marks are checked."""

    from prism_infer import _native

    lib = _native.device_lib(q.device)
    offsets = torch.tensor(cu, dtype=torch.int32, device="cuda")
    batch, (tokens, heads, dim), kv_heads = len(cu) - 1, q.shape, k.shape[1]
    need = lib.prism_prompt_attention_workspace_bytes(batch, tokens, k.shape[0], heads, kv_heads, dim)
    (all_out, out), (all_scratch, scratch) = _guarded(q.numel() * 2), _guarded(need)
    out = out.view(q.dtype).view(q.shape)
    rc = lib.prism_prompt_attention(
        q.data_ptr(), _native.strides(q), k.data_ptr(), _native.strides(k), v.data_ptr(), _native.strides(v),
        _native.dtype_code(q.dtype), offsets.data_ptr(), offsets.data_ptr(), out.data_ptr(), _native.strides(out), batch, tokens,
        k.shape[0], heads, kv_heads, dim, dim ** -0.5, scratch.data_ptr() if need else None, need, _native.stream_handle(q.device))
    _native.check(rc, "prompt_attention")
    for whole in (all_out, all_scratch):
        assert (whole[:GUARD] == MARK).all() and (whole[whole.numel() - GUARD:] == MARK).all()
    return out, need


def _inputs(seed, tokens, heads=2, kv_heads=1, dim=64):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(tokens, h, dim, generator=g).to(torch.bfloat16) for h in (heads, kv_heads, kv_heads)]


@pytest.mark.parametrize("batch", [3, 40, 64, 65, 200, 256, 257, 3001])
@pytest.mark.parametrize("tokens", [150, 3000])
def test_sequences_that_share_rows(batch, tokens):
    """Every other sequence has all rows, the ones between go back: far more blocks than the rows allow for."""

    require_gpu()
    q, k, v = (x.cuda() for x in _inputs(1, tokens))
    _, need = _call(q, k, v, [tokens * (i % 2) for i in range(batch + 1)])
    assert (need > 0) == (batch <= 256 and tokens > 512)


@pytest.mark.parametrize("batch", [20, 64, 65, 130, 256, 257, 900])
def test_sequences_left_out_beside_valid_ones(batch):
    """Offsets that leave the tensors and come back: two sequences left out, the others as they would be alone."""

    require_gpu()
    g = torch.Generator().manual_seed(batch)
    cu, valid = [0], []
    while len(cu) <= batch:
        at = cu[-1]
        if len(cu) % 7 == 3 and len(cu) + 1 <= batch:
            cu += [10**9, at + 2]
            continue
        cu.append(at + int(torch.randint(0, 9, (1,), generator=g)))
        valid.append((at, cu[-1]))
    q, k, v = _inputs(2, cu[-1] + 4)
    out, _ = _call(*(x.cuda() for x in (q, k, v)), cu)
    out = out.cpu()
    for a, b in valid:
        want, bound = attention64(q[a:b], k[a:b], v[a:b], 64 ** -0.5)
        assert_within(out[a:b], want, bound, f"rows {a}..{b}")
    assert (out[cu[-1]:] == 0).all()
