"""Chunks of few rows over 4-bit caches (drafted tokens to check): against the definition, masks, errors, padding, graphs."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _fp4 import Pool, check, chunk_reference
from _helpers import require_gpu
from prism_infer.ops import paged_prefill
from prism_infer.ops.paged_prefill import paged_prefill_attention
from test_gpu_fp4_attention import chunk, queries

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16

CASES = [
    # new tokens, context lengths, heads, kv heads, dim, page, dtype: up to 32 rows (tokens times heads of a kv head) a sequence
    ([5] * 4, [700, 5, 64, 63], 32, 8, 128, 256, BF16),
    ([8, 8], [65, 2000], 16, 4, 128, 64, F16),              # 32 rows
    ([4, 4, 4], [4, 5, 131], 16, 4, 128, 16, BF16),         # 16 rows, a whole block
    ([1, 1], [1, 900], 8, 8, 128, 16, BF16),                # a row
    ([7, 2, 3], [100, 64, 66], 9, 3, 128, 48, F16),         # groups of 3, pages that end inside a step
    ([60] + [1] * 40, [300] + [70] * 40, 8, 2, 128, 16, BF16),  # few on average
    ([2, 1], [513, 300], 32, 2, 128, 32, BF16),             # groups of 16: a token a block
    ([1, 1, 2], [90, 17, 64], 20, 1, 128, 16, F16),         # more heads than a block's rows
    ([6, 3], [150, 40], 8, 2, 64, 16, BF16),
    ([5, 5, 5], [300, 6, 129], 4, 4, 64, 256, F16),
    ([32, 32], [64, 190], 1, 1, 64, 80, BF16),
    ([3] * 130, [20 + 7 * i for i in range(130)], 6, 6, 64, 16, BF16),  # more sequences than lanes
    ([6, 3], [9000, 3], 10, 5, 128, 256, BF16),             # a long one in many parts
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}of{max(c[1])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{str(c[6])[6:]}")
def test_few_rows_match_the_definition(case):
    require_gpu()
    new, ctx, heads, kv_heads, dim, page, dtype = case
    assert sum(new) * heads // kv_heads <= 32 * len(new)
    pool = Pool(ctx, page=page, kv_heads=kv_heads, dim=dim, seed=sum(ctx) + heads)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = queries(cu[-1], heads, dim, dtype, seed=heads + 2)
    out = chunk(pool, q, cu, dim ** -0.5, kv_heads)
    want, bound = chunk_reference(pool, q, cu, dim ** -0.5)
    check(out, want, bound, str(case[2:6]))
    for _ in range(2):
        assert torch.equal(out, chunk(pool, q, cu, dim ** -0.5, kv_heads))


def test_nan_only_where_it_is_seen():
    """A NaN key among the drafted tokens is the later tokens' alone, as is a NaN block of values; the earlier rows are exact."""

    require_gpu()
    pool = Pool([70, 64, 130], page=16, kv_heads=2, dim=128, seed=41)
    cu = [0, 8, 16, 24]
    q = queries(24, 8, 128, BF16, seed=41)
    want, bound = chunk_reference(pool, q, cu, 0.09)
    at = lambda i, t: (int(pool.tables[i, t // 16]), t % 16)  # noqa: E731
    b, r = at(0, 66)                                  # its token 62 + 4
    pool.ks.view(torch.uint8)[b, r, 1, 2] = 255
    b, r = at(1, 61)                                  # its token 56 + 5
    pool.vs.view(torch.uint8)[b, r, 0, 3] = 255
    b, r = at(2, 10)                                  # in front of all of its tokens
    pool.vs.view(torch.uint8)[b, r, 1, 0] = 255
    out = chunk(pool, q, cu, 0.09, 2).cpu()
    nan = torch.zeros(24, 8, 128, dtype=torch.bool)
    nan[4:8, 4:] = True
    nan[8 + 5:16, :4, 96:] = True
    nan[16:, 4:, :32] = True
    assert torch.equal(out.isnan(), nan)
    check(torch.where(nan, 0, out), torch.where(nan, 0, want), bound, "the others")


def test_bytes_of_later_tokens_do_not_matter_to_earlier_ones():
    require_gpu()
    pool = Pool([100], page=16, kv_heads=1, dim=128, seed=42)
    q = queries(8, 4, 128, BF16, seed=42)
    want, bound = chunk_reference(pool, q, [0, 8], 0.09)
    for c, fill in ((pool.kc, 0xFF), (pool.vc, 0xFF), (pool.ks, 254), (pool.vs, 254)):
        c.view(torch.uint8)[int(pool.tables[0, 6]), 0:4] = fill  # tokens 96 to 99: the last four
    # (rows that share a wave with rows that are not finite are summed in another order: the definition's bound, not the same bits)
    check(chunk(pool, q, [0, 8], 0.09, 1)[:4], want[:4], bound[:4], "earlier tokens")


def test_errors_are_those_of_longer_chunks(monkeypatch):
    """Lengths and block ids, by either host path, and rows in front of the first sequence and behind the last."""

    require_gpu()
    pool = Pool([100, 40], page=16, kv_heads=2, dim=128, seed=43)
    q = queries(20, 8, 128, BF16, seed=43)
    want, bound = chunk_reference(pool, q, [3, 9, 13], 0.09)
    bad = {}
    for value in (10 ** 6, -1, pool.kc.shape[0]):
        bad[value] = pool.tables.clone()
        bad[value][1, 1] = value
    for path in range(2):
        if path:
            monkeypatch.setattr(paged_prefill, "_HOST", None)
        got = chunk(pool, q, [3, 9, 13], 0.09, 2)
        assert got.shape[0] == 10
        check(got, want[3:13], bound[3:13], "rows within a larger batch")
        for cu, lens, tables, match in (([0, 0, 16], None, None, "invalid paged prefill lengths: query=0"),
                                        ([0, 6, 4], None, None, "invalid paged prefill lengths"),
                                        ([0, 8, 16], [100, 5], None, "invalid paged prefill lengths"),
                                        ([0, 8, 16], [100, 0], None, "invalid paged prefill lengths"),
                                        ([0, 8, 16], None, bad[10 ** 6], "exceeds cache capacity"),
                                        ([0, 8, 16], None, bad[pool.kc.shape[0]], "exceeds cache capacity"),
                                        ([0, 8, 16], None, bad[-1], "invalid block table")):
            keep = pool.lens.clone()
            if lens is not None:
                pool.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            with pytest.raises(RuntimeError, match=match):
                chunk(pool, q, cu, 0.09, 2, tables=tables)
            pool.lens.copy_(keep)
        assert torch.equal(chunk(pool, q, [3, 9, 13], 0.09, 2), got)


def test_a_captured_check_of_drafts():
    """Replayed with other lengths: padding is zeros, a sequence without rows takes nothing from the others."""

    require_gpu()
    pool = Pool([100, 40, 700], page=16, kv_heads=2, dim=128, seed=44)
    q = queries(24, 8, 128, BF16, seed=44)
    cu = torch.tensor([0, 5, 10, 15], dtype=torch.int32, device="cuda")
    lens = pool.lens.clone()
    context = SimpleNamespace(block_tables=pool.tables, context_lens=lens, cu_seqlens_q=cu)
    call = lambda: paged_prefill_attention(q, pool.kc, pool.vc, context, num_heads=8, num_kv_heads=2, scale=0.09,  # noqa: E731
                                           k_scale_cache=pool.ks, v_scale_cache=pool.vs)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step, ctx in (([0, 5, 10, 15], [100, 40, 700]), ([2, 3, 20, 24], [1, 18, 699]), ([0, 8, 16, 24], [90, 33, 64]), ([0, 1, 2, 3], [1, 1, 1])):
        cu.copy_(torch.tensor(step, dtype=torch.int32))
        lens.copy_(torch.tensor(ctx, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got[step[0]:step[-1]], call())
        assert bool((got[:step[0]] == 0).all()) and bool((got[step[-1]:] == 0).all())
    # a sequence without new tokens, and one whose context is too short: invalid, their neighbours as ever
    cu.copy_(torch.tensor([0, 5, 5, 10], dtype=torch.int32))
    lens.copy_(torch.tensor([100, 40, 700], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone()
    want, bound = chunk_reference(SimpleNamespace(ctx=[100, 700], kc=pool.kc, rows=lambda i: pool.rows([0, 2][i])), q, [0, 5, 10], 0.09)
    check(got[:10], want[:10], bound[:10], "beside a sequence without tokens")
    assert bool((got[10:] == 0).all())
    for step, ctx in (([0, 10, 5, 15], [100, 40, 700]), ([9, 5, 3, 0], [100, 40, 700]), ([-5, 5, 10, 90], [100, 40, 700])):  # out of order
        cu.copy_(torch.tensor(step, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
    cu.copy_(torch.tensor([0, 5, 10, 15], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[:15].clone(), call())


@pytest.mark.parametrize("new", [[1, 1], [5, 3], [60, 44]])
def test_float16_ends_of_the_range(new):
    """Keys and values from float16's smallest to its largest: all exact there, in chunks and one token at a time."""

    require_gpu()
    from _fp4 import decode_reference
    from test_gpu_fp4_attention import decode

    pool = Pool([150, 64], page=16, kv_heads=2, dim=128, seed=45, spread=False)
    g = torch.Generator().manual_seed(45)
    for scales in (pool.ks, pool.vs):  # 0.5 * 2^-23 to 6 * 2^13
        e = scales.view(torch.uint8)
        e.copy_(torch.randint(104, 141, e.shape, generator=g))
    cu = [0, new[0], sum(new)]
    q = queries(cu[-1], 8, 128, F16, seed=45)
    q = q * 2.0 ** -13  # scores of up to a few hundred
    want, bound = chunk_reference(pool, q, cu, 0.09)
    check(chunk(pool, q, cu, 0.09, 2), want, bound, "chunks")
    want, bound = decode_reference(pool, q[:2], 0.09)
    check(decode(pool, q[:2], 0.09), want, bound, "one token")
