"""Decode over 4-bit caches where a workgroup's share of the work is several steps: of one sequence, of a tail, a whole one and a
head, of more sequences than descriptions fit.

Which shares a case has follows from its lengths at 256 CUs (768 shares); the rules are restated here, so that a case that
no longer reaches what it is for fails.
"""

from __future__ import annotations

import pytest
import torch

from _fp4 import BLOCK, E8M0, FP4, VALUES, attend, check
from _helpers import require_gpu
from test_gpu_fp4_attention import decode, queries

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
CUS, SHARES = 256, 768


class RandomPool:
    """Random codes and exponents in scattered pages."""

    def __init__(self, ctx, *, page, kv_heads, dim, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.page = list(ctx), page
        need = [-(-n // page) for n in self.ctx]
        blocks, width = sum(need) + 3, max(need)
        fill = lambda n, low, high: torch.randint(low, high, (blocks, page, kv_heads, n), generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
        self.kc, self.vc = (fill(dim // 2, 0, 256).view(FP4) for _ in range(2))
        self.ks, self.vs = fill(dim // BLOCK, 123, 127).view(E8M0), fill(dim // BLOCK, 122, 131).view(E8M0)
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        tables = torch.full((len(need), width), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            tables[i, :n] = order[at:at + n]
            at += n
        self.tables, self.lens = tables.cuda(), torch.tensor(self.ctx, dtype=torch.int32, device="cuda")

    def rows(self, i):
        """Sequence i's keys and values in 64 bits, on the GPU."""

        t = torch.arange(self.ctx[i], device="cuda")
        where = self.tables[i].long()[t // self.page], t % self.page
        out = []
        for payload, scales in ((self.kc, self.ks), (self.vc, self.vs)):
            p, e = payload.view(torch.uint8)[where].long(), scales.view(torch.uint8)[where].double()
            grid = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64, device="cuda")
            codes = grid[torch.stack([p & 15, p >> 4], -1).flatten(-2)]
            out.append((codes.unflatten(-1, (-1, BLOCK)) * torch.exp2(e - 127)[..., None]).flatten(-2))
        return out


def expected(pool, q, scale):
    q = q.double()
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i, n in enumerate(pool.ctx):
        if n == 0:
            continue
        k, v = pool.rows(i)
        group = q.shape[1] // k.shape[1]
        seen = torch.ones(group, n, dtype=torch.bool, device="cuda")
        for h in range(k.shape[1]):
            rows = slice(h * group, (h + 1) * group)
            out[i, rows], bound[i, rows] = attend(q[i, rows], k[:, h].contiguous(), v[:, h].contiguous(), scale, seen, pool.weight)
    return out.cpu(), bound.cpu()


def division(ctx, heads, kv_heads, dim, page):
    """(steps of a share, entries of the list, row blocks) as the launch has them."""

    at_once = 4 if kv_heads % 4 == 0 else 2 if kv_heads % 2 == 0 else 1
    step, group = 64 * 4 // at_once, heads // kv_heads
    rows = 16 if group > 8 else 8 if group > 4 or dim == 64 else 4
    blocks = kv_heads // at_once * -(-group // rows)
    room = max(-(-n // page) for n in ctx) * page
    whole = room <= 2 * step
    total = blocks * sum(1 if whole else max(-(-n // step), 1) for n in ctx)
    numbers = blocks * len(ctx)
    least = min((total - 1) // CUS, 2) if not whole and total // 4 >= numbers else 0
    return max((total - 1) // SHARES, least) + 1, total, numbers


def lengths(n, top, seed, zeros=0):
    g = torch.Generator().manual_seed(seed)
    ctx = torch.randint(1, top + 1, (n,), generator=g)
    ctx[torch.randperm(n, generator=g)[:zeros]] = 0
    ctx[n // 2] = top
    return ctx.tolist()


CASES = {
    # lengths, heads, kv heads, dim, page, dtype; steps of a share, whether sequences are described by number
    "one of 12000: two steps": ([12000], 32, 8, 128, 256, BF16, 2, True),
    "one of 33500: three steps": ([33500], 32, 8, 128, 256, BF16, 3, True),
    "one of 140000, one head, 64 dims": ([35000 * 4], 8, 1, 64, 64, F16, 3, True),
    "two of 40000, two heads": ([40000, 39999], 8, 2, 128, 16, BF16, 3, True),
    "500 with some empty: more than descriptions": (lengths(500, 400, 1, zeros=40), 32, 8, 128, 16, BF16, 5, False),
    "900 of two heads, some empty": (lengths(900, 700, 2, zeros=50), 8, 2, 128, 64, F16, 4, False),
    "800 of one head": (lengths(800, 1500, 3, zeros=3), 4, 1, 128, 256, BF16, 4, False),
    "450 of groups of 8, 64 dims": (lengths(450, 500, 4, zeros=10), 64, 8, 64, 16, BF16, 5, False),
    "300 of groups of 20, in two blocks": (lengths(300, 600, 5, zeros=5), 40, 2, 128, 32, F16, 3, True),
    "70 of 1 to 40 steps": (lengths(70, 2560, 6, zeros=2), 32, 8, 128, 64, BF16, 4, True),
    "70 of 1 to 40 steps, f16": (lengths(70, 2560, 7), 16, 4, 64, 256, F16, 3, True),
    "110 of two heads": (lengths(110, 5120, 8, zeros=2), 8, 2, 128, 256, BF16, 3, True),
    "100 of one head": (lengths(100, 10240, 9), 16, 1, 128, 64, BF16, 3, True),
    "90 of three heads": (lengths(90, 2600, 10, zeros=1), 12, 3, 128, 16, BF16, 3, True),
}


@pytest.mark.parametrize("name", CASES)
def test_shares_of_several_steps(name):
    require_gpu()
    ctx, heads, kv_heads, dim, page, dtype, share, by_number = CASES[name]
    got_share, total, numbers = division(ctx, heads, kv_heads, dim, page)
    assert (got_share, numbers <= SHARES) == (share, by_number), (got_share, total, numbers)
    pool = RandomPool(ctx, page=page, kv_heads=kv_heads, dim=dim, seed=len(ctx))
    pool.weight = 2.0 ** -8 if dtype == BF16 else 2.0 ** -16
    q = queries(len(ctx), heads, dim, dtype, seed=heads)
    got = decode(pool, q, dim ** -0.5)
    want, bound = expected(pool, q, dim ** -0.5)
    check(got, want, bound, name)
    empty = torch.tensor([n == 0 for n in ctx])
    assert bool((got.cpu()[empty] == 0).all())
    assert torch.equal(got, decode(pool, q, dim ** -0.5))
