"""More tokens than one launch of 2^32 threads holds: up to the limit of 2^31 rows that the entry states, the last like the first."""

from __future__ import annotations

import pytest
import torch

from _fp4 import encode, pack
from _helpers import require_gpu
from test_gpu_rotary_store import make_cache, rotated, same_bytes, table

pytestmark = pytest.mark.gpu
TOKENS = 2 ** 26 + 1001  # a wave each


def test_the_tokens_behind_the_first_launch():
    require_gpu()
    from prism_infer.ops.kv_cache_store import store_kvcache
    from prism_infer.ops.rotary_kv_store import rotate_store_kvcache

    g = torch.Generator(device="cuda").manual_seed(1)
    # token t's row is 64 numbers from 8 t on: 16-byte rows that overlap
    flat = torch.randn(8 * TOKENS + 192, generator=g, device="cuda").bfloat16()
    q, k, v = (flat[64 * i:].as_strided((TOKENS, 1, 64), (8, 64, 1)) for i in range(3))
    edge = (2 ** 32 - 256) // 64
    seen = torch.tensor([0, 1, 77, *range(edge - 4, edge + 5), TOKENS - 2, TOKENS - 1])
    slots = torch.full((TOKENS,), -1, dtype=torch.int32, device="cuda")
    slots[seen.cuda()] = torch.arange(seen.numel(), dtype=torch.int32, device="cuda")
    positions = (torch.arange(TOKENS, device="cuda") % 53).int()
    cos_sin = table(53, 64)
    kc, vc, ks, vs = make_cache("fp4", 1, 16, 1, 64)
    got_q, got_k = rotate_store_kvcache(q, k, v, cos_sin.cuda(), positions, kc, vc, slots, ks, vs, return_key=True)
    want_q, want_k = (rotated(x[seen.cuda()].cpu(), cos_sin, positions[seen.cuda()].cpu()) for x in (q, k))
    assert same_bytes(got_q[seen.cuda()], want_q) and same_bytes(got_k[seen.cuda()], want_k)
    del got_q, got_k
    n = seen.numel()
    for payload, scales, rows in ((kc, ks, want_k), (vc, vs, v[seen.cuda()].cpu())):
        codes, e = encode(rows)
        assert torch.equal(payload.cpu().view(torch.uint8)[0, :n], pack(codes)) and torch.equal(scales.cpu().view(torch.uint8)[0, :n], e)
        assert bool((payload.view(torch.uint8)[0, n:] == 0x55).all())
    # and the store, which has no queries
    kc, vc, ks, vs = make_cache("fp4", 1, 16, 1, 64)
    store_kvcache(k, v, kc, vc, slots, ks, vs)
    codes, e = encode(k[seen.cuda()].cpu())
    assert torch.equal(kc.cpu().view(torch.uint8)[0, :n], pack(codes)) and torch.equal(ks.cpu().view(torch.uint8)[0, :n], e)
