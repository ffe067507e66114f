"""Attention over a 4-bit paged cache on the GPU against the definition in 64 bits."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from _fp4 import Pool, check, chunk_reference, decode_reference
from prism_infer.ops.paged_decode import paged_decode_attention
from prism_infer.ops.paged_prefill import paged_prefill_attention

pytestmark = pytest.mark.gpu


def queries(rows, heads, dim, dtype, seed):
    return torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def decode(pool, q, scale, **more):
    return paged_decode_attention(q, pool.kc, pool.vc, pool.tables, pool.lens, scale, k_scale_cache=pool.ks,
                                  v_scale_cache=pool.vs, **more)


def chunk(pool, q, cu, scale, kv_heads, tables=None):
    context = SimpleNamespace(block_tables=pool.tables if tables is None else tables, context_lens=pool.lens,
                              cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    return paged_prefill_attention(q, pool.kc, pool.vc, context, num_heads=q.shape[1], num_kv_heads=kv_heads, scale=scale,
                                   k_scale_cache=pool.ks, v_scale_cache=pool.vs)


DECODE = [
    # context lengths, heads, kv heads, dim, page, dtype
    ([1], 4, 1, 128, 16, torch.bfloat16),
    ([0, 1, 2, 63, 64, 65], 32, 8, 128, 256, torch.bfloat16),
    ([700], 32, 8, 128, 256, torch.bfloat16),
    ([3000, 1, 0, 129], 8, 2, 128, 64, torch.bfloat16),
    ([257, 255, 256], 16, 4, 128, 16, torch.float16),
    ([100, 513], 64, 8, 128, 256, torch.bfloat16),      # groups of 8
    ([70, 300], 12, 4, 128, 48, torch.bfloat16),        # groups of 3, pages that end inside a tile
    ([70, 300], 8, 8, 128, 16, torch.float16),          # no grouping
    ([129, 31], 16, 1, 128, 32, torch.bfloat16),        # groups of 16
    ([129, 400], 20, 1, 128, 16, torch.float16),        # more rows than a block
    ([65, 190], 36, 2, 128, 112, torch.bfloat16),
    ([5, 1000], 16, 4, 64, 16, torch.float16),
    ([66, 999, 1], 8, 8, 64, 256, torch.bfloat16),
    ([66, 257], 9, 1, 64, 80, torch.bfloat16),
    ([300, 17], 15, 5, 128, 16, torch.bfloat16),        # an odd number of kv heads
    ([9, 210, 64] * 30, 6, 6, 64, 16, torch.bfloat16),  # more sequences than lanes
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{str(c[5])[6:]}")
def test_decode_matches_the_definition(case):
    ctx, heads, kv_heads, dim, page, dtype = case
    pool = Pool(ctx, page=page, kv_heads=kv_heads, dim=dim, seed=sum(ctx) + heads)
    q = queries(len(ctx), heads, dim, dtype, seed=heads)
    out = decode(pool, q, dim ** -0.5)
    want, bound = decode_reference(pool, q, dim ** -0.5)
    check(out, want, bound, str(case[:5]))
    for i, n in enumerate(ctx):
        if n == 0:
            assert bool((out[i] == 0).all())


CHUNKS = [
    # new tokens, context lengths, heads, kv heads, dim, page, dtype
    ([1], [1], 4, 1, 128, 16, torch.bfloat16),
    ([5] * 8, [700, 5, 64, 63, 65, 300, 129, 1000], 32, 8, 128, 256, torch.bfloat16),
    ([17, 1, 64, 200], [17, 90, 500, 201], 8, 2, 128, 16, torch.float16),
    ([130, 3], [400, 70], 12, 4, 128, 48, torch.bfloat16),
    ([70, 129], [70, 700], 4, 4, 64, 64, torch.bfloat16),
    ([33, 2], [100, 40], 9, 1, 64, 16, torch.float16),
    ([300, 260], [900, 260], 32, 8, 128, 256, torch.bfloat16),
    ([2] * 70, [30 + 3 * i for i in range(70)], 2, 1, 128, 16, torch.bfloat16),
]


@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: f"{len(c[0])}x{max(c[0])}of{max(c[1])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{str(c[6])[6:]}")
def test_chunks_match_the_definition(case):
    new, ctx, heads, kv_heads, dim, page, dtype = case
    pool = Pool(ctx, page=page, kv_heads=kv_heads, dim=dim, seed=sum(ctx) + heads)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = queries(cu[-1], heads, dim, dtype, seed=heads + 1)
    out = chunk(pool, q, cu, dim ** -0.5, kv_heads)
    want, bound = chunk_reference(pool, q, cu, dim ** -0.5)
    check(out, want, bound, str(case[2:6]))


@pytest.mark.parametrize("scale", [0.0, -0.3, 30.0])
def test_unusual_scales(scale):
    """A scale of 0 weighs all keys the same, a negative one prefers the other end, a large one a single key."""

    pool = Pool([100, 300], page=64, kv_heads=2, dim=128, seed=4, spread=False)
    q = queries(2, 8, 128, torch.bfloat16, seed=4)
    want, bound = decode_reference(pool, q, scale)
    check(decode(pool, q, scale), want, bound, f"scale {scale}")
    q = queries(30, 8, 128, torch.bfloat16, seed=4)
    want, bound = chunk_reference(pool, q, [0, 10, 30], scale)
    check(chunk(pool, q, [0, 10, 30], scale, 2), want, bound, f"chunk scale {scale}")


def test_queries_of_wide_range():
    """Values from 2^-30 to 2^6 in one row, and a tiny row."""

    pool = Pool([200, 64], page=16, kv_heads=2, dim=128, seed=6)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(2, 8, 128, generator=g) * torch.exp2(torch.randint(-30, 7, (2, 8, 128), generator=g).float())
    q[1, 3] = 0
    q[1, 4] *= 1e-30
    q = q.to(torch.bfloat16).cuda()
    want, bound = decode_reference(pool, q, 0.1)
    check(decode(pool, q, 0.1), want, bound, "wide range")


def test_missing_blocks_and_bounds():
    """Blocks of -1 and behind the cache are skipped; max_context_len and the table's width bound the keys."""

    pool = Pool([300, 130, 64, 200], page=16, kv_heads=2, dim=128, seed=8)
    tables = pool.tables.clone()
    tables[0, 3], tables[0, 7], tables[0, 8] = -1, 10**6, -5
    tables[2] = -1
    pool.tables = tables
    q = queries(4, 8, 128, torch.bfloat16, seed=8)
    want, bound = decode_reference(pool, q, 0.09)
    out = decode(pool, q, 0.09)
    check(out, want, bound, "missing blocks")
    assert bool((out[2] == 0).all())
    limit = torch.tensor(77, dtype=torch.int32, device="cuda")
    want, bound = decode_reference(pool, q, 0.09, limit=77)
    check(decode(pool, q, 0.09, max_context_len=limit), want, bound, "max_context_len")
    pool.lens = torch.tensor([10**9, -5, 64, 200], dtype=torch.int32, device="cuda")
    pool.ctx = [pool.width * 16, 0, 64, 200]
    want, bound = decode_reference(pool, q, 0.09)
    check(decode(pool, q, 0.09), want, bound, "longer than the table")


def test_bytes_behind_the_last_key_do_not_matter():
    """What the last page holds behind the context, NaN exponents included, and pages nobody names."""

    pool = Pool([70, 17, 129], page=32, kv_heads=2, dim=128, seed=10)
    q = queries(3, 8, 128, torch.bfloat16, seed=10)
    first = decode(pool, q, 0.09)
    cu = [0, 7, 8, 20]
    qc = queries(20, 8, 128, torch.bfloat16, seed=11)
    first_chunk = chunk(pool, qc, cu, 0.09, 2)
    used = torch.zeros(pool.kc.shape[0], 32, dtype=torch.bool)
    for i, n in enumerate(pool.ctx):
        for t in range(n):
            used[int(pool.tables[i, t // 32]), t % 32] = True
    for c, fill in ((pool.kc, 0xFF), (pool.vc, 0xFF), (pool.ks, 255), (pool.vs, 255)):
        c.view(torch.uint8)[~used.cuda()] = fill
    assert torch.equal(first, decode(pool, q, 0.09))
    assert torch.equal(first_chunk, chunk(pool, qc, cu, 0.09, 2))


def test_nan_keys_and_values():
    """A NaN key makes the rows that see it NaN; a NaN block of values the dims it covers, in these rows."""

    pool = Pool([100, 100, 100], page=16, kv_heads=2, dim=128, seed=12)
    q = queries(3, 8, 128, torch.bfloat16, seed=12)
    b, r = int(pool.tables[0, 2]), 5
    pool.ks.view(torch.uint8)[b, r, 1, 2] = 255
    b, r = int(pool.tables[1, 6]), 1  # token 97
    pool.vs.view(torch.uint8)[b, r, 0, 3] = 255
    out = decode(pool, q, 0.09)
    nan = torch.zeros(3, 8, 128, dtype=torch.bool)
    nan[0, 4:] = True
    nan[1, :4, 96:] = True
    assert torch.equal(torch.isnan(out.cpu()), nan)
    cu = [0, 50, 90, 100]
    qc = queries(100, 8, 128, torch.bfloat16, seed=13)
    out = chunk(pool, qc, cu, 0.09, 2)
    nan = torch.zeros(100, 8, 128, dtype=torch.bool)
    nan[0:50, 4:] = True           # tokens 50 to 99 see token 37
    nan[50 + 37:90, :4, 96:] = True  # tokens 97 to 99 of 60 to 99
    assert torch.equal(torch.isnan(out.cpu()), nan)


def test_large_and_small_exponents():
    """Values whose exponents span the range of 16-bit results, and keys whose scores they carry."""

    pool = Pool([150, 64], page=16, kv_heads=2, dim=64, seed=14, spread=False)
    e = pool.vs.view(torch.uint8)
    g = torch.Generator().manual_seed(14)
    e.copy_(torch.randint(60, 190, e.shape, generator=g))
    q = queries(2, 4, 64, torch.bfloat16, seed=14)
    want, bound = decode_reference(pool, q, 0.125)
    check(decode(pool, q, 0.125), want, bound, "exponents")


def test_chunk_errors_and_padding():
    pool = Pool([100, 40], page=16, kv_heads=2, dim=128, seed=16)
    q = queries(40, 8, 128, torch.bfloat16, seed=16)
    want, bound = chunk_reference(pool, q, [3, 20, 33], 0.09)
    got = chunk(pool, q, [3, 20, 33], 0.09, 2)
    assert got.shape[0] == 30
    check(got, want[3:33], bound[3:33], "rows within a larger batch")
    with pytest.raises(RuntimeError, match="invalid paged prefill lengths: query=0"):
        chunk(pool, q, [0, 0, 40], 0.09, 2)
    with pytest.raises(RuntimeError, match="invalid paged prefill lengths: query=41|invalid paged prefill lengths"):
        pool.lens[1] = 10
        chunk(pool, q, [0, 20, 40], 0.09, 2)
    pool.lens[1] = 40
    bad = pool.tables.clone()
    bad[1, 1] = 10**6
    with pytest.raises(RuntimeError, match="exceeds cache capacity"):
        chunk(pool, q, [0, 20, 40], 0.09, 2, tables=bad)
    bad[1, 1] = -1
    with pytest.raises(RuntimeError, match="invalid block table"):
        chunk(pool, q, [0, 20, 40], 0.09, 2, tables=bad)


def test_strided_caches_and_queries():
    """Layers of one pool, and queries inside a packed projection."""

    pool = Pool([90, 300], page=16, kv_heads=2, dim=128, seed=18)
    blocks = pool.kc.shape[0]
    layers = []
    for c in (pool.kc, pool.vc, pool.ks, pool.vs):
        big = torch.zeros(blocks, 3, *c.shape[1:], dtype=torch.uint8, device="cuda")
        big[:, 1] = c.view(torch.uint8)
        layers.append(big.view(c.dtype)[:, 1])
    packed = torch.zeros(2, 3 * 8 * 128, dtype=torch.bfloat16, device="cuda")
    q = packed[:, 1024:2048].unflatten(1, (8, 128))
    q.copy_(queries(2, 8, 128, torch.bfloat16, seed=18))
    want = decode(pool, q.contiguous(), 0.09)
    got = paged_decode_attention(q, layers[0], layers[1], pool.tables, pool.lens, 0.09, k_scale_cache=layers[2], v_scale_cache=layers[3])
    assert torch.equal(got, want)
    wide = torch.full((2, 64), -1, dtype=torch.int32, device="cuda")  # a table with a column stride
    wide[:, 0:2 * pool.width:2] = pool.tables
    got = paged_decode_attention(q, layers[0], layers[1], wide[:, 0:2 * pool.width:2], pool.lens, 0.09, k_scale_cache=layers[2],
                                 v_scale_cache=layers[3])
    assert torch.equal(got, want)


def test_split_and_whole_give_the_same_within_the_bound_and_repeat():
    """A long sequence among short ones, twice: the work's division follows the lengths alone."""

    pool = Pool([5000, 3, 77], page=256, kv_heads=4, dim=128, seed=20)
    q = queries(3, 16, 128, torch.bfloat16, seed=20)
    want, bound = decode_reference(pool, q, 128 ** -0.5)
    one = decode(pool, q, 128 ** -0.5)
    check(one, want, bound, "long and short")
    for _ in range(3):
        assert torch.equal(one, decode(pool, q, 128 ** -0.5))


def test_captured_decode_follows_its_lengths():
    pool = Pool([200, 90, 0, 300], page=16, kv_heads=2, dim=128, seed=22)
    q = queries(4, 8, 128, torch.bfloat16, seed=22)
    lens = pool.lens.clone()
    limit = torch.tensor(300, dtype=torch.int32, device="cuda")
    call = lambda: paged_decode_attention(q, pool.kc, pool.vc, pool.tables, lens, 0.09, k_scale_cache=pool.ks,  # noqa: E731
                                          v_scale_cache=pool.vs, max_context_len=limit)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in ([200, 90, 0, 300], [1, 1, 1, 1], [190, 96, 0, 17], [0, 0, 0, 0]):
        lens.copy_(torch.tensor(step, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call()), step
        assert not math.isnan(float(got.float().sum()))


def test_captured_chunks_zero_their_padding():
    pool = Pool([100, 40], page=16, kv_heads=2, dim=128, seed=24)
    q = queries(64, 8, 128, torch.bfloat16, seed=24)
    cu = torch.tensor([0, 20, 33], dtype=torch.int32, device="cuda")
    context = SimpleNamespace(block_tables=pool.tables, context_lens=pool.lens, cu_seqlens_q=cu)
    call = lambda: paged_prefill_attention(q, pool.kc, pool.vc, context, num_heads=8, num_kv_heads=2, scale=0.09,  # noqa: E731
                                           k_scale_cache=pool.ks, v_scale_cache=pool.vs)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in ([0, 20, 33], [0, 40, 64], [5, 6, 7]):
        cu.copy_(torch.tensor(step, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert got.shape[0] == 64
        assert torch.equal(got[step[0]:step[-1]], call())
        assert bool((got[:step[0]] == 0).all()) and bool((got[step[-1]:] == 0).all())


def test_two_streams_at_once():
    pool = Pool([3000, 900], page=256, kv_heads=2, dim=128, seed=26)
    q = queries(2, 8, 128, torch.bfloat16, seed=26)
    want = decode(pool, q, 0.09)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [decode(pool, q, 0.09) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
