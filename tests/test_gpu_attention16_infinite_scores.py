"""Rows whose visible scores are all -inf: the softmax is 0 / 0, NaN; only a row that sees no key is 0.

The definition is written out here in 64 bits (masked scores -inf, exponentials against the row's maximum); finite rows
have the bounds of _attention16.
"""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _attention16 import assert_within, attention64, offsets
from _helpers import require_gpu

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _definition(q, k, v, scale):
    n, m, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    for j in range(n):
        last = m - n + j
        if last < 0:
            continue
        for h in range(q.shape[1]):
            scores = k[:last + 1, h // group].double() @ q[j, h].double() * scale
            w = torch.exp(scores - scores.max())
            out[j, h] = (w / w.sum()) @ v[:last + 1, h // group].double()
    return out


def _check(got, q, k, v, cu_q, cu_k, scale):
    got, nans, empty = got.cpu(), 0, 0
    for i in range(len(cu_q) - 1):
        rows, keys = slice(cu_q[i], cu_q[i + 1]), slice(cu_k[i], cu_k[i + 1])
        want = _definition(q[rows], k[keys], v[keys], scale)
        _, bound = attention64(q[rows], k[keys], v[keys], scale)
        nans += int(want.isnan().any(-1).sum())
        empty += int((want == 0).all(-1).sum())
        assert_within(got[rows], want, bound, f"sequence {i}")
    return nans, empty


def _inputs(seed, tokens_q, tokens_k, heads, kv_heads, dim, dtype):
    """Every key has a negative dim 3, so that a query that is infinite there scores -inf everywhere."""

    g = torch.Generator().manual_seed(seed)
    q = torch.randn(tokens_q, heads, dim, generator=g).to(dtype)
    k, v = (torch.randn(tokens_k, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    k[:, :, 3] = -k[:, :, 3].abs() - 0.5
    return q, k, v


def _prompt(q, k, v, cu_q, cu_k, scale):
    from prism_infer.ops.prompt_attention import prompt_attention

    cq, ck = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cu_q, cu_k))
    return prompt_attention(q.cuda(), k.cuda(), v.cuda(), cq, num_heads=q.shape[1], num_kv_heads=k.shape[1], scale=scale,
                            cu_seqlens_k=ck)


# (query lengths, key lengths, heads, kv heads): whole blocks; blocks of many parts beside rows without a key; about as
# many blocks as CUs, each by two groups of waves
SHAPES = [([40, 9, 70], [40, 4, 200], 4, 2), ([3, 5, 2], [6000, 2, 2500], 4, 1), ([10, 1000], [4, 1600], 32, 8)]


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("lq,lk,heads,kv_heads", SHAPES[:2])
def test_infinite_queries_and_keys(lq, lk, heads, kv_heads, dtype, dim):
    require_gpu()
    cu_q, cu_k = offsets(lq), offsets(lk)
    q, k, v = _inputs(3, cu_q[-1], cu_k[-1], heads, kv_heads, dim, dtype)
    q[1, 0, 3] = q[cu_q[-1] - 1, heads - 1, 3] = float("inf")
    # a first key that every query scores -inf: the first row sees nothing else
    q[cu_q[1]:cu_q[2], :, 7] = q[cu_q[1]:cu_q[2], :, 7].abs() + 0.5
    k[cu_k[1], 0, 7] = float("-inf")
    nans, empty = _check(_prompt(q, k, v, cu_q, cu_k, dim ** -0.5), q, k, v, cu_q, cu_k, dim ** -0.5)
    assert nans >= 3 and empty >= 2 * heads  # (rows before their keys see none)


def test_two_groups_of_waves():
    require_gpu()
    lq, lk, heads, kv_heads = SHAPES[2]
    cu_q, cu_k = offsets(lq), offsets(lk)
    q, k, v = _inputs(4, cu_q[-1], cu_k[-1], heads, kv_heads, 128, BF16)
    rows = [(cu_q[-1] - 1, 0), (cu_q[1] + 300, 9), (cu_q[1], 31)]
    for row, head in rows:
        q[row, head, 3] = float("inf")
    got = _prompt(q, k, v, cu_q, cu_k, 0.1).cpu()
    want = torch.zeros(got.shape[:2], dtype=torch.bool)
    for row, head in rows:
        want[row, head] = True
    assert torch.equal(got.isnan().all(-1), want) and torch.equal(got.isnan().any(-1), want)
    assert (got[:6] == 0).all()  # rows before their keys


@pytest.mark.parametrize("page,dtype,lens", [(16, F16, [(5, 70), (1, 1)]), (64, BF16, [(2, 5000), (3, 900)])])
def test_over_pages(page, dtype, lens):
    require_gpu()
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    cu_q, cu_k = offsets([n for n, _ in lens]), offsets([m for _, m in lens])
    q, k, v = _inputs(5, cu_q[-1], cu_k[-1], 4, 2, 128, dtype)
    q[0, 1, 3] = q[cu_q[1], 2, 3] = float("inf")
    counts = [-(-m // page) for _, m in lens]
    tables = torch.full((len(lens), max(counts)), -1, dtype=torch.int32)
    caches = [torch.zeros(sum(counts), page, 2, 128, dtype=dtype) for _ in range(2)]
    at = 0
    for i, n in enumerate(counts):
        tables[i, :n] = torch.arange(at, at + n, dtype=torch.int32)
        for cache, rows in zip(caches, (k, v)):
            cache[at:at + n].view(-1, 2, 128)[:lens[i][1]] = rows[cu_k[i]:cu_k[i + 1]]
        at += n
    context = SimpleNamespace(block_tables=tables.cuda(), context_lens=torch.tensor([m for _, m in lens], dtype=torch.int32, device="cuda"),
                              cu_seqlens_q=torch.tensor(cu_q, dtype=torch.int32, device="cuda"))
    got = paged_prefill_attention(q.cuda(), caches[0].cuda(), caches[1].cuda(), context, num_heads=4, num_kv_heads=2, scale=0.09)
    assert _check(got, q, k, v, cu_q, cu_k, 0.09)[0] == 2
