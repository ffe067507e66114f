"""Rows behind the last key hold anything, exponents that float16 does not hold among them: not a bit of the output changes, as no
block takes its slow walk for them."""

from __future__ import annotations

import pytest
import torch

from _fp4 import Pool
from _helpers import require_gpu
from test_gpu_fp4_attention import chunk, decode, queries
from test_gpu_fp4_chunk_range import offsets

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.mark.parametrize("exponent", [2, 60, 103, 141, 200, 254, 255])
@pytest.mark.parametrize("new,ctx,heads,kv_heads,dim,page", [([7, 1, 12], [70, 17, 129], 8, 2, 128, 256), ([7, 1, 12], [70, 17, 129], 8, 2, 128, 32),
                                                             ([40, 3], [200, 1000], 4, 2, 64, 64), ([40, 3], [199, 1001], 4, 2, 64, 16),
                                                             ([600], [1505], 16, 8, 128, 256), ([500], [1203], 16, 8, 64, 48)])
def test_rows_behind_the_last_key(new, ctx, heads, kv_heads, dim, page, exponent):
    require_gpu()
    pool = Pool(ctx, page=page, kv_heads=kv_heads, dim=dim, seed=10)
    q, cu = queries(sum(new), heads, dim, F16, seed=11), offsets(new)
    first = chunk(pool, q, cu, 0.09, kv_heads)
    one = decode(pool, q[:len(ctx)], 0.09)
    used = torch.zeros(pool.kc.shape[0], page, dtype=torch.bool)
    for i, n in enumerate(pool.ctx):
        for t in range(n):
            used[int(pool.tables[i, t // page]), t % page] = True
    for c, fill in ((pool.kc, 0x75), (pool.vc, 0x75), (pool.ks, exponent), (pool.vs, exponent)):
        c.view(torch.uint8)[~used.cuda()] = fill
    assert torch.equal(first, chunk(pool, q, cu, 0.09, kv_heads))
    assert torch.equal(one, decode(pool, q[:len(ctx)], 0.09))
