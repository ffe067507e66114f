"""Decode over 4-bit caches whose values reach the end of bf16: finite outputs from them are finite, whatever lies beside them."""

from __future__ import annotations

import pytest
import torch

from _fp4 import Pool, check, decode_reference
from _helpers import require_gpu
from test_gpu_fp4_attention import decode, queries

pytestmark = pytest.mark.gpu
GEOMETRIES = [(32, 8, 128, 256), (8, 2, 128, 16), (16, 1, 128, 64), (8, 8, 64, 16), (12, 1, 64, 48)]


def lost(pool, q):
    """Weights end at 2^-126, and beside values of 2^81 and more they are 2^-32 times exp(score - max): 2^-94 of the largest
    weight, times |v|, may be missing from a row's output (whose sum of weights is at least 1)."""

    out = torch.zeros(q.shape, dtype=torch.float64)
    for i in range(q.shape[0]):
        _, v, _ = pool.rows(i)
        out[i] = 2.0 ** -94 * v.abs().sum(0).repeat_interleave(q.shape[1] // v.shape[1], 0)
    return out


@pytest.mark.parametrize("low,high", [(247, 252), (252, 252), (200, 215), (100, 252)])
@pytest.mark.parametrize("geometry", GEOMETRIES, ids=lambda c: "-".join(map(str, c)))
def test_values_at_the_end_of_the_range(geometry, low, high):
    """Exponent bytes up to 252: 6 * 2^125 is below bf16's largest number.  Growing scores raise the running max step by step."""

    require_gpu()
    heads, kv_heads, dim, page = geometry
    pool = Pool([300, 65, 1, 700], page=page, kv_heads=kv_heads, dim=dim, seed=heads + dim, spread=False)
    e = pool.vs.view(torch.uint8)
    e.copy_(torch.randint(low, high + 1, e.shape, generator=torch.Generator().manual_seed(low)))
    for scale in (dim ** -0.5, 8 * dim ** -0.5):
        q = queries(4, heads, dim, torch.bfloat16, seed=low)
        want, bound = decode_reference(pool, q, scale)
        check(decode(pool, q, scale), want, bound + lost(pool, q), f"bytes {low} to {high}, scale {scale:.3f}")


def test_large_values_in_some_parts_of_a_long_sequence():
    require_gpu()
    pool = Pool([6000, 900], page=16, kv_heads=2, dim=128, seed=3, spread=False)
    e, table = pool.vs.view(torch.uint8), pool.tables.cpu()
    e[int(table[0, 100])] = 250
    e[int(table[0, 300]), 5, 1, 2] = 252
    e[int(table[1, 20]), :, 0] = 249
    q = queries(2, 8, 128, torch.bfloat16, seed=3)
    want, bound = decode_reference(pool, q, 0.09)
    check(decode(pool, q, 0.09), want, bound + lost(pool, q), "large values here and there")


def test_nan_values_beside_large_ones():
    """A NaN block is the dims it covers, the others are as ever; zeros of large blocks are zeros."""

    require_gpu()
    pool = Pool([200, 64], page=16, kv_heads=2, dim=128, seed=5, spread=False)
    e, table = pool.vs.view(torch.uint8), pool.tables.cpu()
    e.fill_(251)
    pool.vc.view(torch.uint8)[..., :16] = 0  # the first 32 dims
    q = queries(2, 8, 128, torch.bfloat16, seed=5)
    want, bound = decode_reference(pool, q, 0.09)
    e[int(table[0, 3]), 2, 1, 3] = 255
    got = decode(pool, q, 0.09).cpu()
    nan = torch.zeros(2, 8, 128, dtype=torch.bool)
    nan[0, 4:, 96:] = True
    assert torch.equal(got.isnan(), nan) and bool((got[..., :32] == 0).all())
    check(torch.where(nan, 0, got), torch.where(nan, 0, want), bound, "the others")
