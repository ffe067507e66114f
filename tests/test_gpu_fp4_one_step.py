"""Decode over 4-bit caches whose tables hold a few steps of keys a sequence, split or not, and few or many sequences."""

from __future__ import annotations

import pytest
import torch

from _fp4 import Pool, check, decode_reference
from _helpers import require_gpu
from test_gpu_fp4_attention import decode, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,page,top", [(32, 8, 16, 64), (8, 2, 64, 128), (4, 1, 256, 256), (20, 1, 16, 255), (32, 8, 16, 65), (8, 2, 64, 129),
                                                     (32, 8, 64, 128), (8, 2, 64, 256), (4, 1, 256, 512), (32, 8, 16, 129), (8, 2, 64, 257), (4, 1, 16, 600)])
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


@pytest.mark.parametrize("heads,kv_heads,page,dim", [(4, 1, 64, 128), (8, 2, 32, 128), (6, 3, 128, 64), (4, 1, 48, 128), (8, 2, 16, 64), (8, 4, 16, 128)])
def test_missing_blocks_by_heads_and_pages(heads, kv_heads, page, dim):
    """Blocks below 0 and behind the cache are left out, whatever share of a step a page is."""

    require_gpu()
    pool = Pool([5 * page + 7, 3 * page, 20 * page - 1], page=page, kv_heads=kv_heads, dim=dim, seed=page)
    pool.tables[0, 1], pool.tables[0, 4], pool.tables[1, :3], pool.tables[2, 19] = -1, pool.kc.shape[0], 2 ** 31 - 1, -5
    q = queries(3, heads, dim, torch.bfloat16, seed=page)
    want, bound = decode_reference(pool, q, 0.1)
    got = decode(pool, q, 0.1)
    check(got, want, bound, "missing blocks")
    assert bool((got[1] == 0).all())
