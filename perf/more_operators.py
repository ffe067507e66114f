"""Performance cases of the 4-bit paged cache and of what writes into any cache, each with its plain form beside the
framework's entry point.

* ``rotate``: position rotation of a step's queries and keys, the keys and values appended to a paged cache on the way
  (``rotate_store_kvcache``), over caches of 16 bits, scaled FP8 and 4 bits; what a 4-bit cache then holds of the step is
  read back as 16-bit rows (``load_kvcache``).
* ``decode4``: decode attention over a 4-bit paged cache (``paged_decode_attention``).
* ``chunk4``: attention of a chunk of new tokens over a 4-bit paged cache (``paged_prefill_attention``).

A 4-bit cache holds E2M1 values, two a byte, with one power of two (E8M0) per token, KV head and 32 dims: the smallest
one at which the block's largest magnitude is at most 7 of it, so that rounding to +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}, ties
to the even code, is off by half a step at most.

The geometry is the repository's: 32 query heads over 8 KV heads and its tensor-parallel shards, head_dim 128, pages of
256 tokens scattered over a pool; other groups, head_dim 64 and pages of 16 as its tests have them.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

_PACKAGE = str(Path(__file__).resolve().parents[1] / "prism-infer_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
FP4_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FP4_BLOCK = 32
FP8_MOST, FP8_FLOOR = 448.0, 1.0e-6


def listed() -> list:
    return [
        # the smallest step: one user's next token, 16-bit cache
        {"name": "rotate_one_16", "kind": "rotate", "tokens": 1, "pad": 0, "q_heads": 32, "heads": 8, "dim": 128,
         "rotary": 128, "pairs": False, "axes": 1, "dtype": "bf16", "cache": "16", "page": 256, "positions": 40960},
        # the decode step of a loaded server, scaled FP8 cache
        {"name": "rotate_decode_64_fp8", "kind": "rotate", "tokens": 64, "pad": 0, "q_heads": 32, "heads": 8, "dim": 128,
         "rotary": 128, "pairs": False, "axes": 1, "dtype": "bf16", "cache": "fp8", "page": 256, "positions": 40960},
        # a mixed prefill batch of a smaller float16 model, half of each head rotated by neighbouring pairs, padded rows
        {"name": "rotate_pairs_777_fp4", "kind": "rotate", "tokens": 777, "pad": 64, "q_heads": 16, "heads": 4, "dim": 64,
         "rotary": 32, "pairs": True, "axes": 1, "dtype": "f16", "cache": "fp4", "page": 16, "positions": 8192},
        # a long prompt with images, whose tokens have three positions each
        {"name": "rotate_axes_8192_fp4", "kind": "rotate", "tokens": 8192, "pad": 0, "q_heads": 32, "heads": 8, "dim": 128,
         "rotary": 128, "pairs": False, "axes": 3, "dtype": "bf16", "cache": "fp4", "page": 256, "positions": 40960},
        # one user's conversation
        {"name": "decode4_one_1800", "kind": "decode4", "batch": 1, "min_len": 1800, "max_len": 1800, "q_heads": 32,
         "heads": 8, "dim": 128, "dtype": "bf16", "page": 256, "pad": 0},
        # ragged conversations of a smaller float16 model over small pages, rows padded for a captured step
        {"name": "decode4_ragged_f16", "kind": "decode4", "batch": 13, "min_len": 1, "max_len": 2000, "q_heads": 16,
         "heads": 4, "dim": 64, "dtype": "f16", "page": 16, "pad": 3},
        # the mixed step of a loaded server
        {"name": "decode4_mixed_64", "kind": "decode4", "batch": 64, "min_len": 1024, "max_len": 16380, "q_heads": 32,
         "heads": 8, "dim": 128, "dtype": "bf16", "page": 256, "pad": 0},
        # long documents
        {"name": "decode4_long_16", "kind": "decode4", "batch": 16, "min_len": 32768, "max_len": 32768, "q_heads": 32,
         "heads": 8, "dim": 128, "dtype": "bf16", "page": 256, "pad": 0},
        # a few drafted tokens of each of eight conversations, checked in one step
        {"name": "chunk4_draft_8x5", "kind": "chunk4", "batch": 8, "min_len": 5, "max_len": 5, "min_prefix": 700,
         "max_prefix": 4090, "q_heads": 32, "heads": 8, "dim": 128, "dtype": "bf16", "page": 256},
        # users' next messages behind long cached conversations
        {"name": "chunk4_hit_12000", "kind": "chunk4", "batch": 2, "min_len": 90, "max_len": 240, "min_prefix": 12000,
         "max_prefix": 12000, "q_heads": 32, "heads": 8, "dim": 128, "dtype": "bf16", "page": 256},
        # ragged chunks on a tensor-parallel shard, small pages, float16
        {"name": "chunk4_page16_f16", "kind": "chunk4", "batch": 12, "min_len": 1, "max_len": 300, "min_prefix": 0,
         "max_prefix": 2000, "q_heads": 16, "heads": 4, "dim": 128, "dtype": "f16", "page": 16},
        # the largest: chunked prefill far into four long prompts
        {"name": "chunk4_long_4", "kind": "chunk4", "batch": 4, "min_len": 2048, "max_len": 2048, "min_prefix": 8192,
         "max_prefix": 8192, "q_heads": 32, "heads": 8, "dim": 128, "dtype": "bf16", "page": 256},
    ]


def _log_uniform(rng, low, high) -> int:
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng) -> dict:
    while True:
        kind = rng.choice(["rotate", "decode4", "chunk4"])
        q_heads, heads = rng.choice([(32, 8), (32, 8), (16, 4), (8, 2), (4, 1), (64, 8), (8, 8), (12, 4)])
        case = {"kind": kind, "q_heads": q_heads, "heads": heads, "dtype": rng.choice(["bf16", "bf16", "f16"]),
                "dim": rng.choice([128, 128, 64]), "page": rng.choice([256, 256, 64, 16])}
        if kind == "rotate":
            case |= {"tokens": _log_uniform(rng, 1, 8192), "pad": rng.choice([0, 0, 64]), "pairs": rng.random() < 0.25,
                     "rotary": rng.choice([case["dim"], case["dim"], case["dim"] // 2]), "axes": rng.choice([1, 1, 3]),
                     "cache": rng.choice(["16", "fp8", "fp4", "fp4"]), "positions": rng.choice([8192, 40960])}
        elif kind == "decode4":
            max_len = _log_uniform(rng, 1, 32768)
            case |= {"batch": _log_uniform(rng, 1, 64), "max_len": max_len,
                     "min_len": max(1, int(max_len * rng.uniform(0.03, 1.0))), "pad": rng.choice([0, 0, 3])}
        else:
            max_len, max_prefix = _log_uniform(rng, 1, 2048), _log_uniform(rng, 50, 12000)
            case |= {"batch": _log_uniform(rng, 1, 16), "max_len": max_len,
                     "min_len": max(1, int(max_len * rng.uniform(0.03, 1.0))), "max_prefix": max_prefix,
                     "min_prefix": int(max_prefix * rng.uniform(0.0, 1.0))}
        w = work(case)
        if w["flops"] <= 1.2e12 and w["bytes"] <= 5.6e8:
            return case


# ---------------------------------------------------------------- sizes that follow from the case alone

def _spread(case, what) -> list:
    low, high = case[f"min_{what}"], case[f"max_{what}"]
    r = random.Random(f"{case['kind']} {what} {case['batch']} {low} {high}")
    return [r.randint(low, high) for _ in range(case["batch"])]


def _rows(case) -> int:
    """Token rows of a rotation step: the step's, padded to a multiple of ``pad``."""

    n, pad = case["tokens"], case["pad"]
    return -(-n // pad) * pad if pad else n


def work(case) -> dict:
    q_heads, heads, dim = case["q_heads"], case["heads"], case["dim"]
    four = heads * (dim // 2 + dim // FP4_BLOCK)  # bytes of a token's keys, or values, in a 4-bit cache
    if case["kind"] == "rotate":
        rows, n = _rows(case), case["tokens"]
        cached = {"16": heads * dim * 2, "fp8": heads * (dim + 4), "fp4": four}[case["cache"]]
        data = rows * 2 * dim * (2 * q_heads) + n * 2 * dim * 2 * heads + n * 2 * cached
        data += min(n, case["positions"]) * case["rotary"] * 4 + rows * 4 * (case["axes"] + 1)
        if case["cache"] == "fp4":
            data += n * 2 * cached + rows * 2 * 2 * dim * heads + rows * 4
        return {"bytes": data, "flops": rows * (q_heads + heads) * case["rotary"] * 3}
    if case["kind"] == "decode4":
        lens = _spread(case, "len")
        index = 4 * len(lens) + 4 * sum(-(-n // case["page"]) for n in lens)
        return {"bytes": sum(lens) * 2 * four + (len(lens) + case["pad"]) * 4 * q_heads * dim + index,
                "flops": 4 * dim * q_heads * sum(lens)}
    new, prefix = _spread(case, "len"), _spread(case, "prefix")
    keys = sum(new) + sum(prefix)
    index = 4 * (2 * case["batch"] + 1) + 4 * sum(-(-(n + p) // case["page"]) for n, p in zip(new, prefix))
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, prefix))
    return {"bytes": 4 * dim * sum(new) * q_heads + keys * 2 * four + index, "flops": 4 * dim * q_heads * pairs}


# ---------------------------------------------------------------- the formats

def _fp4_table(device):
    """The two values of each byte: the low four bits hold the even dim."""

    values = torch.tensor(FP4_VALUES, device=device)
    values = torch.cat([values, -values])
    return torch.stack([values.repeat(16), values.repeat_interleave(16)], dim=1)


def _fp4_encode(x):
    """fp32 [..., dim] -> (bytes [..., dim / 2], exponent bytes [..., dim / 32])."""

    blocks = x.unflatten(-1, (-1, FP4_BLOCK))
    mantissa, exponent = torch.frexp(blocks.abs().amax(-1))  # the mantissa is in [0.5, 1)
    exponent = torch.where(mantissa > 0.875, exponent - 2, exponent - 3).clamp(min=-126)
    exponent = torch.where(mantissa == 0, -126, exponent)
    a = torch.ldexp(blocks.abs(), -exponent[..., None])
    codes = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    codes = (codes + 8 * torch.signbit(blocks)).to(torch.uint8).flatten(-2)
    return codes[..., 0::2] + 16 * codes[..., 1::2], (exponent + 127).to(torch.uint8)


def _fp4_decode(payload, scales):
    """Bytes [..., dim / 2] and exponent bytes [..., dim / 32] -> fp32 [..., dim]."""

    values = _fp4_table(payload.device)[payload.long()].flatten(-2)
    scale = torch.ldexp(torch.ones((), device=payload.device), scales.to(torch.int32) - 127)
    return (values.unflatten(-1, (-1, FP4_BLOCK)) * scale[..., None]).flatten(-2)


# ---------------------------------------------------------------- inputs

def _gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    x = SimpleNamespace(**{**case, "scale": case["dim"] ** -0.5})
    return _prepare_rotate(case, seed, x) if case["kind"] == "rotate" else _prepare_attention(case, seed, x)


def _channels(heads, dim, g):
    """Keys have channels that are larger than others."""

    return torch.exp(0.5 * torch.randn(heads, dim, generator=g, device="cuda"))


def _prepare_rotate(case, seed, x):
    g, rows, n = _gen(seed), _rows(case), case["tokens"]
    dtype = DTYPES[case["dtype"]]
    # q, k and v are views of the packed projection's rows
    qkv = torch.randn(rows, (x.q_heads + 2 * x.heads) * x.dim, generator=g, device="cuda")
    qkv[:, x.q_heads * x.dim:(x.q_heads + x.heads) * x.dim] *= _channels(x.heads, x.dim, g).flatten()
    q, k, v = qkv.to(dtype).split([x.q_heads * x.dim, x.heads * x.dim, x.heads * x.dim], dim=1)
    x.q, x.k, x.v = q.unflatten(1, (x.q_heads, x.dim)), k.unflatten(1, (x.heads, x.dim)), v.unflatten(1, (x.heads, x.dim))
    # the model's table of cosines and sines, with the angles in 64 bits
    half = x.rotary // 2
    rates = 1.0e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angles = torch.arange(x.positions, dtype=torch.float64, device="cuda")[:, None] * rates
    x.table = torch.cat([angles.cos(), angles.sin()], dim=1).float()
    # a decode step's tokens are anywhere, a prompt's follow each other; images' tokens have a row and a column besides
    first = int(torch.randint(0, max(1, x.positions - n), (1,), generator=_gen(seed, "cpu")))
    places = (torch.randint(0, x.positions, (n,), generator=g, device="cuda") if n <= 256
              else first + torch.arange(n, device="cuda") % (x.positions - first))
    positions = torch.zeros(x.axes, rows, dtype=torch.int32, device="cuda")
    positions[:, :n] = places
    if x.axes > 1:
        positions[1:, :n] = (positions[1:, :n] + torch.randint(0, 64, (x.axes - 1, n), generator=g, device="cuda")).clamp(max=x.positions - 1)
    x.place = positions if x.axes > 1 else positions[0]
    x.which = (torch.arange(half, device="cuda") % 3).to(torch.int32) if x.axes > 1 else None
    pages = -(-n // x.page) + 8
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(rows, device="cuda")
    x.slots = torch.where(at < n, order[(at // x.page).clamp(max=pages - 1)] * x.page + at % x.page, -1).to(torch.int32)
    shape = (pages, x.page, x.heads)
    if x.cache == "16":
        x.kc, x.vc = (torch.randn(*shape, x.dim, generator=g, device="cuda").to(dtype) for _ in range(2))
        x.ks = x.vs = None
    elif x.cache == "fp8":
        x.kc, x.vc = (torch.randn(*shape, x.dim, generator=g, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
        x.ks, x.vs = (torch.rand(*shape, generator=g, device="cuda") for _ in range(2))
    else:
        x.kc, x.vc = (torch.randint(0, 256, (*shape, x.dim // 2), generator=g, device="cuda", dtype=torch.uint8)
                      .view(torch.float4_e2m1fn_x2) for _ in range(2))
        x.ks, x.vs = (torch.randint(120, 130, (*shape, x.dim // FP4_BLOCK), generator=g, device="cuda", dtype=torch.uint8)
                      .view(torch.float8_e8m0fnu) for _ in range(2))
    return x


def _prepare_attention(case, seed, x):
    g, dtype = _gen(seed), DTYPES[case["dtype"]]
    new = _spread(case, "len")
    if case["kind"] == "decode4":
        ctx = new + [0] * case["pad"]
        rows = len(ctx)
    else:
        ctx = [n + p for n, p in zip(new, _spread(case, "prefix"))]
        rows = sum(new)
    counts = torch.tensor([-(-n // x.page) for n in ctx])
    pool, width = int(counts.sum()) + 8, int(counts.max())
    column = torch.arange(width)
    tables = torch.full((len(ctx), width), -1, dtype=torch.int32)
    tables[column < counts[:, None]] = torch.randperm(pool, generator=_gen(seed, "cpu"))[:int(counts.sum())].to(torch.int32)
    x.tables, x.ctx = tables.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda")
    x.most, x.most_new = max(ctx), max(new)
    x.cu = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    x.context = SimpleNamespace(block_tables=x.tables, context_lens=x.ctx, cu_seqlens_q=x.cu)
    x.max_ctx = torch.tensor(x.most, dtype=torch.int32, device="cuda")
    x.q = torch.randn(rows, x.q_heads, x.dim, generator=g, device="cuda").to(dtype)
    keys = torch.randn(pool, x.page, x.heads, x.dim, generator=g, device="cuda") * _channels(x.heads, x.dim, g)
    kc, ks = _fp4_encode(keys)
    vc, vs = _fp4_encode(torch.randn(keys.shape, generator=g, device="cuda"))
    x.kc, x.vc = kc.view(torch.float4_e2m1fn_x2), vc.view(torch.float4_e2m1fn_x2)
    x.ks, x.vs = ks.view(torch.float8_e8m0fnu), vs.view(torch.float8_e8m0fnu)
    return x


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return {"rotate": _own_rotate, "decode4": _own_decode, "chunk4": _own_chunk}[state.kind](state)
    return {"rotate": _plain_rotate, "decode4": _plain_decode, "chunk4": _plain_chunk}[state.kind](state)


def _own_rotate(s):
    from prism_infer.ops.kv_cache_load import load_kvcache
    from prism_infer.ops.rotary_kv_store import rotate_store_kvcache

    q = rotate_store_kvcache(s.q, s.k, s.v, s.table, s.place, s.kc, s.vc, s.slots, s.ks, s.vs, position_axes=s.which,
                             interleaved=s.pairs)
    if s.cache == "16":
        return {"q": q, "k": s.kc, "v": s.vc}
    if s.cache == "fp8":
        return {"q": q, "k": s.kc, "v": s.vc, "k_scale": s.ks, "v_scale": s.vs}
    k, v = load_kvcache(s.kc, s.vc, s.slots, s.ks, s.vs, dtype=s.q.dtype)
    return {"q": q, "k": k, "v": v}


def _own_decode(s):
    from prism_infer.ops.paged_decode import paged_decode_attention

    return paged_decode_attention(s.q, s.kc, s.vc, s.tables, s.ctx, s.scale, k_scale_cache=s.ks, v_scale_cache=s.vs,
                                  max_context_len=s.max_ctx)


def _own_chunk(s):
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    return paged_prefill_attention(s.q, s.kc, s.vc, s.context, num_heads=s.q_heads, num_kv_heads=s.heads, scale=s.scale,
                                   k_scale_cache=s.ks, v_scale_cache=s.vs)


def _rotated(x, cos, sin, pairs):
    """The first dims of x [rows, heads, dim], two for each angle, turned; in 32 bits, each product rounded."""

    n = 2 * cos.shape[-1]
    turn, rest = x[..., :n].float(), x[..., n:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if pairs else turn.chunk(2, dim=-1)
    c, s = cos[:, None], sin[:, None]
    first, second = a * c - b * s, b * c + a * s
    turn = torch.stack([first, second], dim=-1).flatten(-2) if pairs else torch.cat([first, second], dim=-1)
    return torch.cat([turn.to(x.dtype), rest], dim=-1)


def _plain_rotate(s):
    half = s.rotary // 2
    rows = s.place[s.which.long()].t() if s.which is not None else s.place[:, None]  # [tokens, half or 1]
    at = torch.arange(half, device="cuda")
    cos, sin = s.table[rows.long(), at], s.table[rows.long(), at + half]
    q, k = _rotated(s.q, cos, sin, s.pairs), _rotated(s.k, cos, sin, s.pairs)
    live = s.slots >= 0
    slots, k, v = s.slots[live].long(), k[live], s.v[live]
    if s.cache == "16":
        s.kc.flatten(0, 1)[slots] = k
        s.vc.flatten(0, 1)[slots] = v
        return {"q": q, "k": s.kc, "v": s.vc}
    if s.cache == "fp8":
        ks, vs = ((t.float().abs().amax(-1) / FP8_MOST).clamp(min=FP8_FLOOR) for t in (k, v))
        s.ks.flatten(0, 1)[slots], s.vs.flatten(0, 1)[slots] = ks, vs
        k8, v8 = ((t.float() / c[..., None]).clamp(-FP8_MOST, FP8_MOST).to(torch.float8_e4m3fn) for t, c in ((k, ks), (v, vs)))
        s.kc.view(torch.uint8).flatten(0, 1)[slots] = k8.view(torch.uint8)
        s.vc.view(torch.uint8).flatten(0, 1)[slots] = v8.view(torch.uint8)
        return {"q": q, "k": s.kc, "v": s.vc, "k_scale": s.ks, "v_scale": s.vs}
    caches = [t.view(torch.uint8).flatten(0, 1) for t in (s.kc, s.ks, s.vc, s.vs)]
    caches[0][slots], caches[1][slots] = _fp4_encode(k.float())
    caches[2][slots], caches[3][slots] = _fp4_encode(v.float())
    held_k, held_v = torch.zeros_like(s.k), torch.zeros_like(s.v)
    held_k[live] = _fp4_decode(caches[0][slots], caches[1][slots]).to(s.k.dtype)
    held_v[live] = _fp4_decode(caches[2][slots], caches[3][slots]).to(s.v.dtype)
    return {"q": q, "k": held_k, "v": held_v}


def _dense(s):
    """Every sequence's keys and values in 32 bits, [batch, heads, tokens of the longest, dim]."""

    at = torch.arange(s.most, device="cuda")
    rows = s.tables[:, at // s.page].clamp(min=0).long() * s.page + at % s.page
    k = _fp4_decode(s.kc.view(torch.uint8).flatten(0, 1)[rows], s.ks.view(torch.uint8).flatten(0, 1)[rows])
    v = _fp4_decode(s.vc.view(torch.uint8).flatten(0, 1)[rows], s.vs.view(torch.uint8).flatten(0, 1)[rows])
    return k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()


def _attend(s, q, seen):
    """q [batch, heads, rows, dim], seen [batch, 1, rows, tokens] -> fp32 [batch, heads, rows, dim]; zeros where nothing is seen."""

    k, v = _dense(s)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * s.scale
    scores = scores.masked_fill_(~seen, -math.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-3.0e38)).exp_()
    return torch.matmul(weights, v) / weights.sum(-1, keepdim=True).clamp(min=1.0e-38)


def _plain_decode(s):
    q = s.q.float().unflatten(1, (s.heads, -1))
    seen = torch.arange(s.most, device="cuda") < s.ctx[:, None, None, None]
    return _attend(s, q, seen).flatten(1, 2).to(s.q.dtype)


def _plain_chunk(s):
    batch, group = s.ctx.numel(), s.q_heads // s.heads
    new = s.cu[1:] - s.cu[:-1]
    token = torch.arange(s.most_new, device="cuda")
    live = token < new[:, None]  # [batch, rows of the longest chunk]
    at = (s.cu[:-1, None] + token).clamp(max=s.q.shape[0] - 1).long()
    q = s.q[at].float().unflatten(2, (s.heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # rows: token, head of the group
    last = (s.ctx - new)[:, None] + token
    seen = torch.arange(s.most, device="cuda") <= last.repeat_interleave(group, 1)[:, None, :, None]
    got = _attend(s, q.contiguous(), seen).unflatten(2, (-1, group)).permute(0, 2, 1, 3, 4)
    return got.reshape(batch, s.most_new, s.q_heads, s.dim)[live].to(s.q.dtype)


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotate(s) if case["kind"] == "rotate" else _exact_attention(s)


def _exact_turn(s, x):
    half, out = s.rotary // 2, x.double().clone()
    for i in range(half):
        place = (s.place if s.which is None else s.place[int(s.which[i])]).long()
        a, b = (2 * i, 2 * i + 1) if s.pairs else (i, i + half)
        z = torch.complex(x[..., a].double(), x[..., b].double())
        z = z * torch.complex(s.table[place, i].double(), s.table[place, i + half].double())[:, None]
        out[..., a], out[..., b] = z.real, z.imag
    return out


def _exact_round4(x):
    """The nearest value of the format, by distance; of two as near the one with the even code."""

    blocks = x.double().unflatten(-1, (-1, FP4_BLOCK))
    most = blocks.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(torch.where(most > 0, most, 1.0) / 7.0)))  # (7 of it is the most)
    grid = torch.tensor(FP4_VALUES, dtype=torch.float64, device=x.device)
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)  # even codes first
    a = (blocks.abs() / scale)
    best, value = torch.full_like(a, math.inf), torch.zeros_like(a)
    for code in order.tolist():
        off = (a - grid[code]).abs()
        value = torch.where(off < best, grid[code], value)
        best = torch.minimum(best, off)
    return (torch.where(most > 0, value * scale, 0.0) * torch.sign(blocks)).flatten(-2)


def _exact_rotate(s):
    q, k = _exact_turn(s, s.q), _exact_turn(s, s.k)
    live = torch.nonzero(s.slots >= 0).flatten()
    slots = s.slots[live].long()
    if s.cache == "fp4":
        held_k, held_v = torch.zeros_like(k), torch.zeros_like(k)
        held_k[live] = _exact_round4(k.to(s.k.dtype))[live]
        held_v[live] = _exact_round4(s.v)[live]
        return {"q": q, "k": held_k, "v": held_v}
    out = {"q": q}
    for name, x, cache, scales in (("k", k, s.kc, s.ks), ("v", s.v.double(), s.vc, s.vs)):
        rows = x[live]
        if s.cache == "fp8":
            rows = rows.to(s.k.dtype).double()
            scale = (rows.abs().amax(-1) / FP8_MOST).clamp(min=FP8_FLOOR)
            rows = rows / scale[..., None]
            out[name + "_scale"] = scales.double()
            out[name + "_scale"].view(-1, s.heads)[slots] = scale
        out[name] = cache.to(torch.float32).double()
        out[name].view(-1, s.heads, s.dim)[slots] = rows
    return out


def _exact_rows(payload, scales, where, h):
    """One head's rows in 64 bits, the values taken apart bit by bit."""

    byte = payload.view(torch.uint8)[where + (h,)].long()
    code = torch.stack([byte % 16, byte // 16], dim=-1).flatten(-2)
    sign, power, bit = 1.0 - 2.0 * (code // 8), code // 2 % 4, code % 2
    size = torch.where(power > 0, (1.0 + 0.5 * bit.double()) * torch.exp2(power.double() - 1.0), 0.5 * bit.double())
    scale = torch.exp2(scales.view(torch.uint8)[where + (h,)].double() - 127.0)
    return sign * size * scale.repeat_interleave(FP4_BLOCK, dim=-1)


def _exact_attention(s):
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    group, ctx, cu = s.q_heads // s.heads, s.ctx.tolist(), s.cu.tolist()
    for i, m in enumerate(ctx):
        a, b = (i, i + 1) if s.kind == "decode4" else (cu[i], cu[i + 1])
        if m == 0:
            continue
        at, n = torch.arange(m, device="cuda"), b - a
        where = (s.tables[i].long()[at // s.page], at % s.page)
        for h in range(s.heads):
            keys, values = _exact_rows(s.kc, s.ks, where, h), _exact_rows(s.vc, s.vs, where, h)
            for j in range(h * group, (h + 1) * group):
                logits = (s.q[a:b, j].double() * s.scale) @ keys.t().contiguous()
                logits[at[None, :] - (m - n) > torch.arange(n, device="cuda")[:, None]] = -math.inf
                out[a:b, j] = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True)) @ values
    return out
