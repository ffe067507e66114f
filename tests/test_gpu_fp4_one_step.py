"""Decode over 4-bit caches whose tables hold one step of keys a sequence: nothing is split, however many sequences there are."""

from __future__ import annotations

import pytest
import torch

from _fp4 import Pool, check, decode_reference
from _helpers import require_gpu
from test_gpu_fp4_attention import decode, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,page,top", [(32, 8, 16, 64), (8, 2, 64, 128), (4, 1, 256, 256), (20, 1, 16, 255), (32, 8, 16, 65), (8, 2, 64, 129)])
@pytest.mark.parametrize("batch", [1, 300])
def test_tables_of_one_step_and_just_more(heads, kv_heads, page, top, batch):
    require_gpu()
    g = torch.Generator().manual_seed(top + batch)
    ctx = torch.randint(0, top + 1, (batch,), generator=g).tolist()
    ctx[0] = top
    pool = Pool(ctx, page=page, kv_heads=kv_heads, dim=128, seed=top)
    q = queries(batch, heads, 128, torch.bfloat16, seed=top)
    want, bound = decode_reference(pool, q, 0.09)
    check(decode(pool, q, 0.09), want, bound, f"{batch} of up to {top}")
