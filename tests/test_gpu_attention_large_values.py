"""Values that reach the end of bf16, over every kind of key: outputs are averages of them, and finite like them.

The values' weighted sum, before it is divided by the weights', can leave fp32.  It is then taken anew with weights of at
most 2^-24: 2^-102 of the row's largest weight, times |v|, may be missing from an output.
"""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _attention16 import assert_within, attention64, offsets
from _fp4 import Pool, check, chunk_reference
from _helpers import require_gpu
from prism_infer.ops.paged_prefill import paged_prefill_attention
from prism_infer.ops.prompt_attention import prompt_attention
from test_gpu_fp4_attention import chunk, queries
from test_gpu_fp4_chunk_range import IDS, SHAPES

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("low,high", [(247, 252), (252, 252), (180, 200), (100, 252)])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_chunks_over_4bit_caches(shape, low, high):
    """Exponent bytes up to 252: 6 * 2^125 is below bf16's largest number."""

    require_gpu()
    new, ctx, heads, kv_heads, dim, page = shape
    pool = Pool(ctx, page=page, kv_heads=kv_heads, dim=dim, seed=9, spread=False)
    e = pool.vs.view(torch.uint8)
    e.copy_(torch.randint(low, high + 1, e.shape, generator=torch.Generator().manual_seed(low)))
    q, cu = queries(sum(new), heads, dim, BF16, seed=9), offsets(new)
    want, bound = chunk_reference(pool, q, cu, dim ** -0.5)
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        bound[a:b] += 2.0 ** -102 * pool.rows(i)[1].abs().sum(0).repeat_interleave(heads // kv_heads, 0)
    check(chunk(pool, q, cu, dim ** -0.5, kv_heads), want, bound, f"bytes {low} to {high}")


def rows(n, heads, dim, seed, power=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=g).clamp(-3.5, 3.5)
    return (x.double() * 2.0 ** power).to(BF16)


@pytest.mark.parametrize("power", [126, 120, 62])
@pytest.mark.parametrize("lens,heads,kv_heads,dim", [([300, 1, 70], 8, 2, 128), ([1500], 16, 8, 128), ([900, 200], 4, 4, 64)])
def test_prompts_and_pages_of_16_bits(lens, heads, kv_heads, dim, power):
    require_gpu()
    n, cu = sum(lens), offsets(lens)
    q, k, v = rows(n, heads, dim, 1), rows(n, kv_heads, dim, 2), rows(n, kv_heads, dim, 3, power)
    want, bound = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    for a, b in zip(cu, cu[1:]):
        want[a:b], bound[a:b] = attention64(q[a:b], k[a:b], v[a:b], dim ** -0.5)
        bound[a:b] += 2.0 ** -102 * v[a:b].double().abs().sum(0).repeat_interleave(heads // kv_heads, 0)
    cu_gpu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu_gpu, num_heads=heads, num_kv_heads=kv_heads, scale=dim ** -0.5)
    assert_within(got, want, bound, "packed")
    for page in (16, 64):
        blocks = [-(-m // page) for m in lens]
        caches = [torch.zeros(sum(blocks), page, kv_heads, dim, dtype=BF16) for _ in range(2)]
        tables = torch.zeros(len(lens), max(blocks), dtype=torch.int32)
        for i, (a, b) in enumerate(zip(cu, cu[1:])):
            first = sum(blocks[:i])
            tables[i, :blocks[i]] = torch.arange(first, first + blocks[i])
            for cache, x in zip(caches, (k, v)):
                cache[first:first + blocks[i]].view(-1, kv_heads, dim)[:b - a] = x[a:b]
        context = SimpleNamespace(block_tables=tables.cuda(), context_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), cu_seqlens_q=cu_gpu)
        got = paged_prefill_attention(q.cuda(), caches[0].cuda(), caches[1].cuda(), context, num_heads=heads, num_kv_heads=kv_heads,
                                      scale=dim ** -0.5)
        assert_within(got, want, bound, f"pages of {page}")
