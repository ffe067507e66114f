"""A prefill step with a request that has no new tokens: taken without a cached prefix, refused with one."""

from __future__ import annotations

import pytest
import torch

from _attention16 import assert_within, attention64
from _helpers import require_gpu

pytestmark = pytest.mark.gpu


def test_requests_without_new_tokens():
    require_gpu()
    from prism_infer.engine.prefill_attention import PagedKVPrefillAttention
    from prism_infer.engine.step_metadata import build_step_metadata

    g = torch.Generator().manual_seed(1)
    layer = PagedKVPrefillAttention(4, 2, 128, 0.1)
    layer.k_cache, layer.v_cache = (torch.zeros(12, 16, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, k, v = (torch.randn(30, h, 128, generator=g).to(torch.bfloat16) for h in (4, 2, 2))
    tables, free = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), torch.arange(12, dtype=torch.int32, device="cuda")
    none, new = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([20, 0, 10], dtype=torch.int32, device="cuda")
    m = build_step_metadata(tables, none, new, block_size=16, num_tokens=30, free_blocks=free).check()
    got = layer(q.cuda(), k.cuda(), v.cuda(), m, cached_prefix=False)
    for a, b in ((0, 20), (20, 30)):
        assert_within(got[a:b], *attention64(q[a:b], k[a:b], v[a:b], 0.1), f"rows {a}..{b}")
    for _ in range(2):
        with pytest.raises(RuntimeError, match="invalid paged prefill lengths: query=0 context=0"):
            layer(q.cuda(), k.cuda(), v.cuda(), m, cached_prefix=True)
