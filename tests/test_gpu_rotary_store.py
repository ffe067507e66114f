"""Rotation with append on the GPU against the definition: bit for bit, as the ops in turn give it.

Every step of the operator is defined to the last bit (fp32 products and sums rounded one by one, one rounding to the
input's type, the store's own bytes), so nothing here has a tolerance but the test against the angles in 64 bits.
"""

from __future__ import annotations

import math

import pytest
import torch

from _fp4 import E8M0, FP4, decode, empty_cache, encode, pack
from prism_infer.ops.kv_cache_load import load_kvcache
from prism_infer.ops.kv_cache_store import _quantize_rows, store_kvcache
from prism_infer.ops.rotary_kv_store import rotate_store_kvcache

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def table(positions, rotary, base=1.0e4):
    half = rotary // 2
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat([angles.cos(), angles.sin()], 1).float()


def rotated(x, cos_sin, positions, axes=None, pairs=False):
    """fp32 on the host, each product and sum rounded, then to x's type."""

    n = cos_sin.shape[1]
    half = n // 2
    at = positions[None].expand(half, -1).t() if axes is None else positions[axes.long()].t()  # [tokens, half]
    i = torch.arange(half).expand_as(at)
    good = (at >= 0) & (at < cos_sin.shape[0])
    safe = at.clamp(0, max(cos_sin.shape[0] - 1, 0)).long()
    c = torch.where(good, cos_sin[safe, i], math.nan)[:, None]
    s = torch.where(good, cos_sin[safe, i + half], math.nan)[:, None]
    t = x[..., :n].float()
    a, b = (t[..., 0::2], t[..., 1::2]) if pairs else (t[..., :half], t[..., half:])
    first, second = a * c - b * s, b * c + a * s
    t = torch.stack([first, second], -1).flatten(-2) if pairs else torch.cat([first, second], -1)
    return torch.cat([t.to(x.dtype), x[..., n:]], -1)


def same_bytes(a, b):
    a, b = a.cpu().contiguous(), b.cpu().contiguous()
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def make(tokens, q_heads, heads, dim, dtype, seed, pad=0):
    """Views of a packed projection."""

    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, (q_heads + 2 * heads) * dim + pad, generator=g)
    qkv[torch.rand(qkv.shape, generator=g) < 0.01] *= 20
    qkv = qkv.to(dtype).cuda()
    q, k, v, _ = qkv.split([q_heads * dim, heads * dim, heads * dim, pad], 1)
    return q.unflatten(1, (q_heads, dim)), k.unflatten(1, (heads, dim)), v.unflatten(1, (heads, dim)), g


def make_cache(kind, blocks, page, heads, dim):
    if kind == "fp4":
        (kc, ks), (vc, vs) = empty_cache((blocks, page, heads, dim)), empty_cache((blocks, page, heads, dim))
        return kc, vc, ks, vs
    dtype = {"fp8": FP8, "fp8_unit": FP8, "bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[kind]
    kc, vc = (torch.full((blocks, page, heads, dim), 0.5, device="cuda").to(dtype) for _ in range(2))
    if kind == "fp8":
        return kc, vc, torch.full((blocks, page, heads), 0.25, device="cuda"), torch.full((blocks, page, heads), 0.25, device="cuda")
    return kc, vc, None, None


def stored(rows, kind, dtype):
    """(payload bytes, scale) of rows, by the store's definition on the host."""

    rows = rows.cpu()
    if kind == "fp4":
        codes, e = encode(rows)
        return pack(codes), e
    if kind == "fp8":
        payload, scale = _quantize_rows(rows, FP8)
        return payload.view(torch.uint8), scale
    return rows.float().to(dtype), None


CASES = [
    # tokens, q heads, kv heads, dim, rotary, pairs, axes, input, cache, row padding
    (1, 32, 8, 128, 128, False, 1, torch.bfloat16, "bf16", 0),
    (64, 32, 8, 128, 128, False, 1, torch.bfloat16, "fp8", 0),
    (5, 32, 8, 128, 128, False, 3, torch.bfloat16, "fp4", 0),
    (600, 32, 8, 128, 128, False, 3, torch.bfloat16, "fp4", 64),
    (513, 4, 1, 128, 64, True, 1, torch.float16, "fp4", 0),
    (37, 12, 3, 64, 64, False, 1, torch.float16, "f16", 8),
    (515, 3, 3, 64, 32, True, 2, torch.float16, "fp4", 0),
    (9, 8, 2, 256, 128, False, 4, torch.float32, "fp8", 0),
    (700, 8, 2, 256, 256, False, 1, torch.float32, "bf16", 0),
    (11, 4, 2, 128, 128, True, 1, torch.bfloat16, "fp8_unit", 0),
    (17, 4, 2, 128, 128, False, 1, torch.bfloat16, "f32", 0),
    # what the vector kernel does not take: other head dims, angles in odd places, rows off 16 bytes
    (21, 4, 2, 96, 96, False, 1, torch.bfloat16, "fp4", 0),
    (21, 4, 2, 32, 32, False, 3, torch.float32, "fp4", 0),
    (13, 3, 1, 80, 20, False, 1, torch.float16, "fp8", 0),
    (13, 3, 1, 128, 26, True, 2, torch.bfloat16, "fp4", 3),
    (7, 5, 5, 48, 48, True, 1, torch.bfloat16, "bf16", 1),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_rotation_and_append_match_the_definition(case):
    tokens, q_heads, heads, dim, rotary, pairs, axes, dtype, kind, pad = case
    q, k, v, g = make(tokens, q_heads, heads, dim, dtype, seed=tokens + dim, pad=pad)
    page = 16
    blocks = -(-tokens // page) + 3
    caches = make_cache(kind, blocks, page, heads, dim)
    before = [None if t is None else t.clone() for t in caches]
    cos_sin = table(2000, rotary)
    positions = torch.randint(0, 2000, (axes, tokens), generator=g, dtype=torch.int32)
    which = torch.randint(0, axes, (rotary // 2,), generator=g, dtype=torch.int32) if axes > 1 else None
    slots = torch.randperm(blocks * page, generator=g)[:tokens].to(torch.int32)
    slots[1::7] = -1
    if tokens > 2:
        slots[2] = blocks * page  # behind the cache
    got_q, got_k = rotate_store_kvcache(
        q, k, v, cos_sin.cuda(), (positions if axes > 1 else positions[0]).cuda(), caches[0], caches[1], slots.cuda(),
        caches[2], caches[3], position_axes=None if which is None else which.cuda(), interleaved=pairs, return_key=True)
    place = positions if axes > 1 else positions[0]
    want_q, want_k = (rotated(x.cpu(), cos_sin, place, which, pairs) for x in (q, k))
    assert same_bytes(got_q, want_q) and got_q.is_contiguous()
    assert same_bytes(got_k, want_k)
    live = (slots >= 0) & (slots < blocks * page)
    at = slots[live].long()
    for rows, payload, scale, old, old_scale in ((want_k, caches[0], caches[2], before[0], before[2]),
                                                 (v.cpu(), caches[1], caches[3], before[1], before[3])):
        data, s = stored(rows[live], kind, payload.dtype)
        flat = old.cpu().contiguous().view(torch.uint8).view(blocks * page, heads, -1).clone()
        flat[at] = data.view(torch.uint8).view(data.shape[0], heads, -1)
        assert torch.equal(payload.cpu().view(torch.uint8).view(blocks * page, heads, -1), flat)
        if s is not None:
            flat = old_scale.cpu().view(torch.uint8).view(blocks * page, heads, -1).clone()
            flat[at] = s.contiguous().view(torch.uint8).view(s.shape[0], heads, -1)
            assert torch.equal(scale.cpu().view(torch.uint8).view(blocks * page, heads, -1), flat)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp4"])
def test_the_same_as_the_two_ops_in_turn(kind):
    q, k, v, g = make(130, 8, 2, 128, torch.bfloat16, seed=3)
    cos_sin, positions = table(4000, 128).cuda(), torch.randint(0, 4000, (130,), generator=g, dtype=torch.int32).cuda()
    slots = torch.randperm(256, generator=g)[:130].to(torch.int32).cuda()
    one, two = make_cache(kind, 16, 16, 2, 128), make_cache(kind, 16, 16, 2, 128)
    _, turned = rotate_store_kvcache(q, k, v, cos_sin, positions, one[0], one[1], slots, one[2], one[3], return_key=True)
    store_kvcache(turned, v.contiguous(), two[0], two[1], slots, two[2], two[3])
    for a, b in zip(one, two):
        assert (a is None and b is None) or same_bytes(a, b)


def test_angles_of_far_positions():
    """The table holds the angles' cosines and sines; the result is within their roundings of the rotation in 64 bits."""

    positions = torch.tensor([0, 1, 131071, 99999], dtype=torch.int32)
    q, k, v, _ = make(4, 4, 2, 128, torch.float32, seed=5)
    cos_sin = table(131072, 128, 1.0e6)
    kc, vc, _, _ = make_cache("f32", 1, 16, 2, 128)
    got = rotate_store_kvcache(q, k, v, cos_sin.cuda(), positions.cuda(), kc, vc, torch.arange(4, dtype=torch.int32, device="cuda"))
    half = 64
    angle = positions.double()[:, None] * 1.0e6 ** (-torch.arange(half, dtype=torch.float64) / half)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = q.cpu().double()[..., :half], q.cpu().double()[..., half:]
    want = torch.cat([a * c - b * s, b * c + a * s], -1)
    # table entry, product and sum: three roundings of 2^-24 of at most |a| + |b| each
    limit = 3 * 2.0 ** -24 * torch.cat([a.abs() + b.abs()] * 2, -1) * (1 + 2.0 ** -20)
    assert bool(((got.cpu().double() - want).abs() <= limit).all())


def test_positions_outside_the_table_are_nan():
    q, k, v, _ = make(6, 4, 2, 128, torch.bfloat16, seed=9)
    cos_sin = table(50, 64)
    positions = torch.tensor([0, 49, 50, -1, 2**31 - 1, 7], dtype=torch.int32)
    kc, vc, ks, vs = make_cache("fp4", 1, 16, 2, 128)
    slots = torch.arange(6, dtype=torch.int32, device="cuda")
    got = rotate_store_kvcache(q, k, v, cos_sin.cuda(), positions.cuda(), kc, vc, slots, ks, vs)
    want = rotated(q.cpu(), cos_sin, positions)
    bad = torch.tensor([False, False, True, True, True, False])
    assert torch.equal(torch.isnan(got.cpu()).any(-1), bad[:, None].expand(6, 4))
    assert torch.equal(torch.nan_to_num(got.cpu().float(), 9.0), torch.nan_to_num(want.float(), 9.0))
    # blocks with a rotated dim are NaN in the cache, the others as ever; values are untouched by it
    assert torch.equal(ks.view(torch.uint8).cpu()[0, :6, :, :2] == 255, bad[:, None, None].expand(6, 2, 2))
    assert bool((ks.view(torch.uint8)[0, :6, :, 2:] != 255).all()) and bool((vs.view(torch.uint8)[0, :6] != 255).all())
    # an axis that is none of the rows
    axes = torch.zeros(32, dtype=torch.int32)
    axes[3], axes[4] = 1, -1
    got = rotate_store_kvcache(q[:2], k[:2], v[:2], cos_sin.cuda(), positions[None, :2].contiguous().cuda(), kc, vc, slots[:2], ks, vs,
                               position_axes=axes.cuda())
    lost = torch.zeros(128, dtype=torch.bool)
    lost[[3, 4, 35, 36]] = True
    assert torch.equal(torch.isnan(got.cpu()), lost.expand(2, 4, 128))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_fp4_store_of_special_rows(dtype, dim):
    """Zeros of either sign, ties, limits between exponents, the largest and smallest values, infinities and NaN."""

    top = torch.finfo(dtype).max
    rows = torch.zeros(12, 1, dim)
    rows[1] = -0.0
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 7.0])
    rows[2, 0, :16] = ties
    rows[3, 0, :32] = torch.tensor([7.0, 6.99, -7.0, 3.5] * 8)
    rows[4, 0, :32] = torch.tensor([7.03125, 0.5, -0.25, 1.0] * 8)
    rows[5, 0, 0] = top
    rows[6, 0, 5] = torch.finfo(dtype).tiny
    rows[7, 0, 6] = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # the smallest subnormal
    rows[8, 0, 3] = math.inf
    rows[9, 0, 40 % dim] = -math.inf
    rows[10, 0, 33 % dim] = math.nan
    rows[11] = torch.randn(dim, generator=torch.Generator().manual_seed(1)) * 1e-6
    rows = rows.to(dtype)
    (kc, ks), (vc, vs) = empty_cache((1, 16, 1, dim)), empty_cache((1, 16, 1, dim))
    store_kvcache(rows.cuda(), -rows.cuda(), kc, vc, torch.arange(12, dtype=torch.int32, device="cuda"), ks, vs)
    for x, payload, scale in ((rows, kc, ks), (-rows, vc, vs)):
        codes, e = encode(x)
        assert torch.equal(scale.cpu().view(torch.uint8)[0, :12], e)
        assert torch.equal(payload.cpu().view(torch.uint8)[0, :12], pack(codes))
        assert bool((payload.cpu().view(torch.uint8)[0, 12:] == 0x55).all())


def test_every_bf16_value_rounds_as_defined():
    """All finite bf16 values, each beside a largest value that fixes its block's exponent."""

    bits = torch.arange(0, 0x7F80, dtype=torch.int32)
    x = bits.to(torch.int16).view(torch.bfloat16).float()
    rows = torch.zeros(x.numel(), 2, BLOCK_DIM)
    rows[:, 0, 0] = x
    rows[:, 1, 1] = -x
    rows[:, 1, 0] = x * 1.75
    rows = rows.to(torch.bfloat16)
    rows = torch.where(torch.isfinite(rows), rows, 0.0)
    n = rows.shape[0]
    (kc, ks), (vc, vs) = empty_cache((n, 16, 2, BLOCK_DIM)), empty_cache((n, 16, 2, BLOCK_DIM))
    slots = (torch.arange(n, device="cuda", dtype=torch.int32) * 16)
    store_kvcache(rows.cuda(), rows.cuda(), kc, vc, slots, ks, vs)
    codes, e = encode(rows)
    assert torch.equal(ks.cpu().view(torch.uint8)[:, 0], e)
    assert torch.equal(kc.cpu().view(torch.uint8)[:, 0], pack(codes))
    assert same_bytes(kc, vc)


BLOCK_DIM = 64


@pytest.mark.parametrize("kind", ["fp4", "fp8", "fp8_unit", "bf16", "f16", "f32"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_load_reads_what_the_slots_hold(kind, dtype):
    _, k, v, g = make(50, 3, 3, 64, torch.bfloat16, seed=21)
    kc, vc, ks, vs = make_cache(kind, 6, 16, 3, 64)
    slots = torch.randperm(96, generator=g)[:50].to(torch.int32).cuda()
    store_kvcache(k.contiguous(), v.contiguous(), kc, vc, slots, ks, vs)
    ask = torch.cat([slots[:20], torch.tensor([-1, 96, 2**31 - 1], dtype=torch.int32, device="cuda"), slots[:1]])
    got = load_kvcache(kc, vc, ask, ks, vs, dtype=dtype)
    for out, cache, scale in zip(got, (kc, vc), (ks, vs)):
        assert out.shape == (24, 3, 64) and out.dtype == dtype
        flat = decode(cache, scale) if kind == "fp4" else cache.float().cpu()
        if kind == "fp8":
            flat = flat * scale.cpu()[..., None]
        flat = flat.float().view(96, 3, 64).to(dtype)
        want = flat[slots[:20].long().cpu()]
        assert same_bytes(out[:20], want) and same_bytes(out[23], want[0])
        assert bool((out[20:23] == 0).all())


def test_fp4_load_of_special_exponents():
    kc, ks = empty_cache((1, 16, 1, 64), fill=0x72)
    e = ks.view(torch.uint8)
    e[0, 0], e[0, 1], e[0, 2], e[0, 3] = 0, 255, 1, 253
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    got, _ = load_kvcache(kc, kc, slots, ks, ks, dtype=torch.float32)
    want = decode(kc, ks)[0, :4].float()
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.cpu(), 0.0), torch.nan_to_num(want, 0.0))


def test_empty_and_padded_calls():
    q, k, v, _ = make(3, 4, 2, 128, torch.bfloat16, seed=2)
    cos_sin = table(10, 128).cuda()
    kc, vc, ks, vs = make_cache("fp4", 1, 16, 2, 128)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    out = rotate_store_kvcache(q[:0], k[:0], v[:0], cos_sin, none, kc, vc, none, ks, vs)
    assert out.shape == (0, 4, 128)
    before = kc.clone()
    pad = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = rotate_store_kvcache(q, k, v, cos_sin, zero, kc, vc, pad, ks, vs)
    assert same_bytes(out, q) and same_bytes(kc, before)  # position 0 turns nothing
    key, value = load_kvcache(kc, vc, none, ks, vs)
    assert key.shape == (0, 2, 128) and value.shape == (0, 2, 128)


def test_captured_steps_follow_their_inputs():
    q, k, v, g = make(16, 8, 2, 128, torch.bfloat16, seed=7)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cos_sin = table(300, 128).cuda()
    positions, slots = torch.arange(16, dtype=torch.int32, device="cuda"), torch.arange(16, dtype=torch.int32, device="cuda")
    kc, vc, ks, vs = make_cache("fp4", 4, 16, 2, 128)
    call = lambda: rotate_store_kvcache(q, k, v, cos_sin, positions, kc, vc, slots, ks, vs)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(3):
        q.copy_(torch.randn(q.shape, generator=g))
        k.copy_(torch.randn(k.shape, generator=g))
        positions.add_(16)
        slots.add_(16)
        graph.replay()
        torch.cuda.synchronize()
        got = (out.clone(), kc.clone(), ks.clone())
        eager = call()
        assert same_bytes(got[0], eager) and same_bytes(got[1], kc) and same_bytes(got[2], ks)


def test_another_stream():
    q, k, v, g = make(40, 8, 2, 128, torch.bfloat16, seed=8)
    cos_sin = table(300, 128).cuda()
    positions = torch.randint(0, 300, (40,), generator=g, dtype=torch.int32).cuda()
    slots = torch.arange(40, dtype=torch.int32, device="cuda")
    one, two = make_cache("fp4", 3, 16, 2, 128), make_cache("fp4", 3, 16, 2, 128)
    want = rotate_store_kvcache(q, k, v, cos_sin, positions, one[0], one[1], slots, one[2], one[3])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = rotate_store_kvcache(q, k, v, cos_sin, positions, two[0], two[1], slots, two[2], two[3])
    side.synchronize()
    assert same_bytes(got, want) and all(same_bytes(a, b) for a, b in zip(one, two))
