"""Chunks over 4-bit caches whose keys and values are no float16 numbers, with float16 queries."""

from __future__ import annotations

import math

import pytest
import torch

from _fp4 import Pool, attend, check, empty_cache
from _helpers import require_gpu
from prism_infer.ops.kv_cache_store import store_kvcache
from test_gpu_fp4_attention import chunk, decode

pytestmark = pytest.mark.gpu
F16 = torch.float16

# new tokens, context lengths, heads, kv heads, dim, page: split keys, two groups of waves, both kinds of pages, both widths
SHAPES = [
    ([5, 3], [700, 65], 32, 8, 128, 256),
    ([40, 2], [300, 90], 8, 2, 128, 16),
    ([7, 20], [3000, 20], 8, 2, 128, 64),
    ([600], [1500], 16, 8, 128, 256),   # two groups
    ([500], [1200], 16, 8, 128, 48),
    ([9, 33], [400, 70], 4, 2, 64, 64),
    ([33, 2], [100, 2000], 9, 1, 64, 16),
    ([600], [1500], 16, 8, 64, 256),
    ([500], [1200], 16, 8, 64, 16),
]
IDS = ["-".join(map(str, [len(s[0]), max(s[0]), max(s[1]), *s[2:]])) for s in SHAPES]


def expected(pool, q, cu, scale, weight=2.0 ** -11):
    """Output and bound: `attend`'s, with scores of up to 256 exact products (a float16 query as the sum of two bf16 numbers,
    the second at most 2^-8 of the first: 136 roundings of 2^-24 of sum |q| |k| beside the 132 that `attend` counts)."""

    q = q.double().cpu()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        k, v, keep = pool.rows(i)
        group = q.shape[1] // k.shape[1]
        seen = keep[None, :] <= (pool.ctx[i] - (b - a) + torch.arange(b - a))[:, None]
        for j in range(q.shape[1]):
            kj, vj = k[:, j // group], v[:, j // group]
            out[a:b, j], bound[a:b, j] = attend(q[a:b, j], kj, vj, scale, seen, weight)
            more = 136 * 2.0 ** -24 * abs(scale) * torch.where(seen, q[a:b, j].abs() @ kj.abs().t(), 0.0).amax(1, keepdim=True)
            w = torch.softmax(torch.where(seen, scale * q[a:b, j] @ kj.t(), -math.inf), 1)
            bound[a:b, j] += 2 * more * (w @ vj.abs())
    return out, bound


def offsets(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def make(shape, low, high):
    """Keys with exponent bytes low to high, and a scale that makes scores of these a few units."""

    new, ctx, heads, kv_heads, dim, page = shape
    pool = Pool(ctx, page=page, kv_heads=kv_heads, dim=dim, seed=sum(ctx), spread=False)
    g = torch.Generator().manual_seed(low)
    e = pool.ks.view(torch.uint8)
    e.copy_(torch.randint(low, high + 1, e.shape, generator=g))
    q = (torch.randn(sum(new), heads, dim, generator=g) * 2.0 ** 8).to(F16)
    return pool, q, 2.0 ** (127 - high) / 2.0 ** 8 / math.sqrt(dim)


@pytest.mark.parametrize("low,high", [(24, 30), (100, 103), (104, 106), (140, 140), (141, 143), (190, 200)])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_keys_beside_float16s_range(shape, low, high):
    require_gpu()
    pool, q, scale = make(shape, low, high)
    want, bound = expected(pool, q, offsets(shape[0]), scale)
    check(chunk(pool, q.cuda(), offsets(shape[0]), scale, shape[3]), want, bound, f"bytes {low} to {high}")


@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_a_few_large_keys(shape, where):
    """Keys that float16 does not hold in one tile of many: their scores are the larger ones, of either sign."""

    require_gpu()
    pool, q, scale = make(shape, 126, 128)
    e, table = pool.ks.view(torch.uint8), pool.tables.cpu()
    for i, n in enumerate(pool.ctx):
        at = {"first": 0, "middle": (n - shape[0][i]) // 2, "last": max(n - shape[0][i] - 1, 0)}[where]
        for t in range(at, min(at + 3, n)):
            e[int(table[i, t // pool.page]), t % pool.page] = 149
    q *= 2.0 ** -18
    scale *= 2.0 ** 18 / 2.0 ** 20
    want, bound = expected(pool, q, offsets(shape[0]), scale)
    check(chunk(pool, q.cuda(), offsets(shape[0]), scale, shape[3]), want, bound, f"large keys: {where}")


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_float16_values_that_are_stored_as_65536(shape):
    """Finite float16 numbers above 57344 are held as 65536, which is finite in decode and in chunks."""

    require_gpu()
    new, ctx, heads, kv_heads, dim, page = shape
    pool = Pool(ctx, page=page, kv_heads=kv_heads, dim=dim, seed=7)
    g = torch.Generator().manual_seed(7)
    rows = pool.kc.shape[0] * page
    k, v = (torch.randn(rows, kv_heads, dim, generator=g).to(F16) for _ in range(2))
    k[::5, :, 3], v[::3, :, 40], v[1::3, :, 40] = 60000.0, 60000.0, -61000.0
    (pool.kc, pool.ks), (pool.vc, pool.vs) = (empty_cache((pool.kc.shape[0], page, kv_heads, dim)) for _ in range(2))
    store_kvcache(k.cuda(), v.cuda(), pool.kc, pool.vc, torch.arange(rows, dtype=torch.int32, device="cuda"), pool.ks, pool.vs)
    q = torch.randn(sum(new), heads, dim, generator=g).to(F16)
    q[:, :, 3] *= 2.0 ** -16
    want, bound = expected(pool, q, offsets(new), 0.1)
    got = chunk(pool, q.cuda(), offsets(new), 0.1, kv_heads).cpu()
    far = want.abs() + bound >= 65504  # (a row that sees one such value alone)
    assert not bool(got.isnan().any()) and bool(got[~far].isfinite().all())
    check(torch.where(far, 0, got), torch.where(far, 0, want), torch.where(far, 0, bound), "chunks")
    for n in range(len(ctx)):  # the last row of each sequence, one token at a time
        want_one, bound_one = want[offsets(new)[n + 1] - 1], bound[offsets(new)[n + 1] - 1]
        one = SimplePool(pool, n)
        got = decode(one, q[offsets(new)[n + 1] - 1][None].cuda(), 0.1)[0]
        check(got, want_one, bound_one, "one token")


class SimplePool:
    """One sequence of a pool."""

    def __init__(self, pool, n):
        self.kc, self.vc, self.ks, self.vs = pool.kc, pool.vc, pool.ks, pool.vs
        self.tables, self.lens = pool.tables[n:n + 1], pool.lens[n:n + 1]


def test_nan_only_where_it_is_seen_beside_small_keys():
    require_gpu()
    pool, q, scale = make(([8, 8], [70, 64], 8, 2, 128, 16), 100, 103)
    cu = [0, 8, 16]
    want, bound = expected(pool, q, cu, scale)
    at = lambda i, t: (int(pool.tables[i, t // 16]), t % 16)  # noqa: E731
    b, r = at(0, 66)
    pool.ks.view(torch.uint8)[b, r, 1, 2] = 255
    b, r = at(1, 61)
    pool.vs.view(torch.uint8)[b, r, 0, 3] = 255
    q[1, 0, 4], q[9, 1, 7] = math.inf, math.nan
    out = chunk(pool, q.cuda(), cu, scale, 2).cpu()
    nan = torch.zeros(16, 8, 128, dtype=torch.bool)
    nan[4:8, 4:] = True
    nan[8 + 5:16, :4, 96:] = True
    nan[1, 0] = nan[9, 1] = True
    assert torch.equal(out.isnan(), nan)
    check(torch.where(nan, 0, out), torch.where(nan, 0, want), bound, "the others")
