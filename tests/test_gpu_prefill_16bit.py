"""GPU paged prefill over bf16 and float16 caches against plain attention in 64 bits (bounds: _attention16)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _attention16 import assert_within, attention64, offsets
from _helpers import require_gpu

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _case(seed, seqs, *, heads=8, kv_heads=2, dim=128, page=64, dtype=BF16, spare=3):
    """Random pages for sequences given as (query_len, context_len); pages and rows in no use hold NaN."""

    g = torch.Generator().manual_seed(seed)
    counts = [-(-ctx // page) for _, ctx in seqs]
    pool = sum(counts) + spare
    perm = torch.randperm(pool, generator=g)
    tables = torch.full((len(seqs), max(counts) + 1), -1, dtype=torch.int32)
    k, v = (torch.full((pool, page, kv_heads, dim), float("nan"), dtype=dtype) for _ in range(2))
    dense, at = [], 0
    for i, (n, (_, ctx)) in enumerate(zip(counts, seqs)):
        ids = perm[at:at + n]
        at += n
        tables[i, :n] = ids.to(torch.int32)
        pair = []
        for cache in (k, v):
            rows = torch.randn(ctx, kv_heads, dim, generator=g).to(dtype)
            for j, b in enumerate(ids.tolist()):
                part = rows[j * page:(j + 1) * page]
                cache[b, :part.shape[0]] = part
            pair.append(rows)
        dense.append(pair)
    cu = offsets([n for n, _ in seqs])
    q = torch.randn(cu[-1], heads, dim, generator=g).to(dtype)
    return SimpleNamespace(q=q, k=k, v=v, tables=tables, lens=[c for _, c in seqs], cu=cu, dense=dense, scale=dim ** -0.5)


def _run(c, **over):
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    x = {n: over.get(n, getattr(c, n)).cuda() for n in ("q", "k", "v", "tables")}
    ctx = SimpleNamespace(block_tables=x["tables"], context_lens=torch.tensor(c.lens, dtype=torch.int32, device="cuda"),
                          cu_seqlens_q=torch.tensor(c.cu, dtype=torch.int32, device="cuda"))
    return paged_prefill_attention(x["q"], x["k"], x["v"], ctx, num_heads=c.q.shape[1], num_kv_heads=c.k.shape[2],
                                   scale=c.scale)


def _want(c):
    parts = [attention64(c.q[a:b], k, v, c.scale) for a, b, (k, v) in zip(c.cu, c.cu[1:], c.dense)]
    return torch.cat([o for o, _ in parts]), torch.cat([b for _, b in parts])


SEQS = [(37, 300), (64, 64), (1, 513), (100, 164), (1, 1), (5, 1000), (33, 33)]


@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 64)])
def test_pages_types_dims(dtype, dim, page):
    require_gpu()
    c = _case(page + dim, SEQS, page=page, dim=dim, dtype=dtype)
    assert_within(_run(c), *_want(c), f"{dtype} {dim} {page}")


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (8, 8), (6, 2), (16, 1), (7, 7), (64, 8)])
def test_groups(heads, kv_heads):
    require_gpu()
    c = _case(heads, [(45, 200), (3, 3), (1, 130), (20, 60)], heads=heads, kv_heads=kv_heads, page=16)
    assert_within(_run(c), *_want(c), f"{heads}/{kv_heads}")


@pytest.mark.parametrize("page,dtype", [(256, BF16), (16, F16)])
def test_short_chunks_behind_long_contexts(page, dtype):
    """One and few tokens behind thousands: few rows, many tiles."""

    require_gpu()
    c = _case(5, [(1, 5000), (4, 3333), (17, 2049)], heads=8, kv_heads=2, page=page, dtype=dtype)
    assert_within(_run(c), *_want(c))


@pytest.mark.parametrize("seqs,heads,kv_heads,dim", [([(1000, 1000)], 32, 8, 128), ([(600, 1003), (520, 700)], 32, 8, 128),
                                                     ([(1001, 1200)], 20, 20, 64)])
@pytest.mark.parametrize("page,dtype", [(64, BF16), (16, F16)])
def test_as_many_blocks_as_cus(page, dtype, seqs, heads, kv_heads, dim):
    require_gpu()
    c = _case(dim + page, seqs, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    assert_within(_run(c), *_want(c))


def test_threads_on_streams_of_their_own():
    """Each thread finds its own outcomes: results of its own lengths, and its own bad table."""

    require_gpu()
    import threading

    cases = [_case(40 + i, [(30 + i, 400 + 90 * i), (5, 60)], page=16) for i in range(4)]
    wants = [_want(c) for c in cases]
    failed, start = [], threading.Barrier(len(cases))

    def work(i):
        try:
            c = cases[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for turn in range(20):
                    if (turn + i) % 5 == 0:
                        tables = c.tables.clone()
                        tables[i % 2, 1] = c.k.shape[0]
                        with pytest.raises((ValueError, RuntimeError, IndexError)):
                            _run(c, tables=tables)
                    else:
                        assert_within(_run(c), *wants[i])
        except BaseException as e:  # noqa: BLE001 (reported by the test's own thread)
            failed.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_large_batch_and_ragged_chunks():
    require_gpu()
    g = torch.Generator().manual_seed(6)
    seqs = [(int(n), int(n + p)) for n, p in zip(torch.randint(1, 30, (100,), generator=g), torch.randint(0, 90, (100,), generator=g))]
    c = _case(7, seqs, page=16)
    assert_within(_run(c), *_want(c))


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("page,dtype", [(256, BF16), (16, F16)])
def test_values_that_are_no_numbers(page, dtype, what):
    require_gpu()
    c = _case(8, [(60, 400), (90, 90)], page=page, dtype=dtype)
    for seq, pos, head, dim in ((0, 370, 1, 3), (1, 50, 0, 77)):
        c.dense[seq][1][pos, head, dim] = float(what)
        c.v[int(c.tables[seq, pos // page]), pos % page, head, dim] = float(what)
    want, bound = _want(c)
    assert not want.isfinite().all() and want.isfinite().any()
    assert_within(_run(c), want, bound)


def test_layouts():
    """Caches as a layer's slice of a pool and with heads before tokens; queries off their 16 bytes."""

    require_gpu()
    c = _case(9, [(30, 100), (5, 70)], page=16)
    want, bound = _want(c)
    pool = torch.stack([c.k, c.v, c.k, c.v]).unflatten(0, (2, 2)).cuda()
    assert_within(_run(c, k=pool[1, 0], v=pool[0, 1]), want, bound, "slices")
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2).cuda() for x in (c.k, c.v)]
    assert_within(_run(c, k=turned[0], v=turned[1]), want, bound, "heads first")
    odd = torch.empty(*c.q.shape[:2], 129, dtype=c.q.dtype, device="cuda")[..., 1:].copy_(c.q)
    assert_within(_run(c, q=odd), want, bound, "odd queries")


def test_pages_behind_two_to_the_31_elements():
    require_gpu()
    c = _case(10, [(20, 80), (7, 40)], page=64, kv_heads=8, heads=8, spare=0)
    far = (2 ** 31) // (64 * 8 * 128) + 5
    k, v = (torch.empty(far + c.k.shape[0], 64, 8, 128, dtype=BF16, device="cuda") for _ in range(2))
    k[far:], v[far:] = c.k.cuda(), c.v.cuda()
    tables = torch.where(c.tables >= 0, c.tables + far, c.tables)
    assert_within(_run(c, k=k, v=v, tables=tables), *_want(c))


@pytest.mark.parametrize("kind,match", [
    ("short_context", "invalid paged prefill lengths: query=30 context=20"),
    ("block_past_cache", "paged KV block id exceeds cache capacity"),
    ("missing_block", "invalid block table for paged KV reference"),
])
def test_errors(kind, match):
    require_gpu()
    c = _case(11, [(10, 40), (30, 300)], page=16)
    if kind == "short_context":
        c.lens[1] = 20
    elif kind == "block_past_cache":
        c.tables[1, 3] = c.k.shape[0] + 5
    else:
        c.tables[1, 5] = -1
    with pytest.raises(RuntimeError, match=match):
        _run(c)
    good = _case(11, [(10, 40), (30, 300)], page=16)
    assert_within(_run(good), *_want(good))


def test_refusals():
    require_gpu()
    c = _case(12, [(4, 20)], page=16)
    with pytest.raises(RuntimeError, match="queries' dtype"):
        _run(c, q=c.q.to(F16))
    with pytest.raises(RuntimeError, match="queries' dtype"):
        _run(c, v=c.v.to(F16))
    small = _case(12, [(4, 20)], page=16, dim=32)
    with pytest.raises(RuntimeError, match="head_dim 64 and 128"):
        _run(small)
    odd = _case(12, [(4, 20)], page=24)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        _run(odd)


def test_captured():
    require_gpu()
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    c = _case(13, [(30, 300), (20, 20), (1, 90)], page=64)
    q, k, v = c.q.cuda(), c.k.cuda(), c.v.cuda()
    ctx = SimpleNamespace(block_tables=c.tables.cuda(), context_lens=torch.tensor(c.lens, dtype=torch.int32, device="cuda"),
                          cu_seqlens_q=torch.tensor(c.cu, dtype=torch.int32, device="cuda"))

    def call():
        return paged_prefill_attention(q, k, v, ctx, num_heads=8, num_kv_heads=2, scale=c.scale)

    eager = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, call()) and torch.equal(out, eager)
