"""4-bit caches and rotation without a GPU: the host's store, shapes and bytes, and every refusal before a launch."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from _fp4 import BLOCK, E8M0, FP4, decode, empty_cache, encode, pack
from prism_infer.engine import kv_quantization as quant
from prism_infer.engine.kv_block_ops import copy_kv_block_prefixes, copy_kv_blocks
from prism_infer.ops.kv_cache_load import load_kvcache
from prism_infer.ops.kv_cache_store import store_kvcache
from prism_infer.ops.paged_decode import paged_decode_attention
from prism_infer.ops.paged_prefill import paged_prefill_attention
from prism_infer.ops.rotary_kv_store import rotate_store_kvcache

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


# ---- the format


def special_rows(dim):
    """Ties, limits of the exponents, zeros, subnormals, the largest values, infinities and NaN."""

    g = torch.Generator().manual_seed(1)
    rows = [torch.randn(dim, generator=g) * 2.0 ** e for e in (-140, -126, -20, 0, 20, 120)]
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.999, 7.0, -0.25, -5.0, -7.0, 0.0, -0.0])
    rows += [steps.repeat(dim // steps.numel() + 1)[:dim] * 2.0 ** e for e in (0, 3, -100)]
    rows.append((torch.full((dim,), 7.0) * (1 + 2.0 ** -23)))  # just above the limit: the next exponent
    rows += [torch.zeros(dim), torch.full((dim,), torch.finfo(torch.float32).max), torch.full((dim,), 2.0 ** -149)]
    for bad in (math.inf, -math.inf, math.nan):
        row = torch.randn(dim, generator=g)
        row[dim // 2 + 3] = bad
        rows.append(row)
    return torch.stack(rows)


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_hosts_store_has_the_formats_bytes(dim, dtype):
    rows = special_rows(dim).to(dtype)[:, None, :].contiguous()
    n = rows.shape[0]
    kc, ks = empty_cache((2, 16, 1, dim), device="cpu")
    vc, vs = empty_cache((2, 16, 1, dim), device="cpu")
    slots = torch.randperm(32, generator=torch.Generator().manual_seed(2))[:n].int()
    slots[1] = -1
    store_kvcache(rows, rows.flip(-1), kc, vc, slots, ks, vs)
    for cache, scales, x in ((kc, ks, rows), (vc, vs, rows.flip(-1))):
        codes, e = encode(x.float())
        payload, exponents = cache.view(torch.uint8).flatten(0, 1), scales.view(torch.uint8).flatten(0, 1)
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                assert torch.equal(payload[s], pack(codes)[i]) and torch.equal(exponents[s], e[i]), (i, x[i])
        untouched = [s for s in range(32) if s not in slots.tolist()]
        assert (payload[untouched] == 0x55).all() and (exponents[untouched] == 127).all()


def test_what_is_stored_is_the_nearest_value():
    """|stored - x| is at most half the grid's step around x (values above 6 units, at most 1 unit, go to 6)."""

    x = torch.randn(64, 2, 128, generator=torch.Generator().manual_seed(3)).double()
    codes, e = encode(x)
    got = decode(pack(codes), e)
    unit = torch.exp2(e.double() - 127).repeat_interleave(BLOCK, -1)
    units = (x / unit).abs()
    step = torch.where(units < 2, 0.5, torch.where(units < 4, 1.0, 2.0))
    assert ((got - x).abs() <= step / 2 * unit).all() and (units <= 7).all()
    smaller = (x / (unit / 2)).abs().unflatten(-1, (-1, BLOCK)).amax(-1)
    assert (smaller > 7).all()  # no smaller exponent would do


def test_shapes_and_bytes():
    assert quant.fp4_payload_shape((3, 16, 2, 128)) == (3, 16, 2, 64)
    assert quant.fp4_scale_cache_shape((3, 16, 2, 64)) == (3, 16, 2, 4)
    for bad in ((3, 16, 2, 80), (2, 64), (3, 0, 2, 64), (3, 16, True, 64)):
        with pytest.raises(ValueError, match="fp4_payload_shape"):
            quant.fp4_payload_shape(bad)
    for bad in ((), (3, 2, 24)):
        with pytest.raises(ValueError, match="fp4_scale_cache_shape"):
            quant.fp4_scale_cache_shape(bad)
    sizes = dict(num_layers=36, page_size=256, num_kv_heads=8, head_dim=128)
    four = quant.kv_block_storage_bytes(**sizes, payload_dtype=FP4, token_head_scales=True)
    assert (four.payload, four.scales) == (9437184, 589824)  # 4.25 bits a value
    full = quant.kv_block_storage_bytes(**sizes, payload_dtype=BF16, token_head_scales=False)
    assert four.total * 16 == full.total * 4.25
    payload, scales = empty_cache((3, 16, 2, 128), device="cpu")
    assert quant.kv_cache_storage_bytes(payload, scales).total == 3 * 16 * 2 * (64 + 4)


def test_blocks_of_a_host_cache_move_with_their_exponents():
    g = torch.Generator().manual_seed(4)
    payload = torch.randint(0, 256, (2, 2, 4, 16, 2, 32), generator=g, dtype=torch.uint8)
    exponent = torch.randint(0, 256, (2, 2, 4, 16, 2, 2), generator=g, dtype=torch.uint8)
    want = [t.clone() for t in (payload, exponent)]
    for t in want:
        t[:, :, 3] = t[:, :, 0]
        t[:, :, 2, :5] = t[:, :, 1, :5]
    copy_kv_blocks(payload.view(FP4), [(0, 3)], exponent.view(E8M0))
    copy_kv_block_prefixes(payload.view(FP4), [(1, 2, 5)], exponent.view(E8M0))
    assert torch.equal(payload, want[0]) and torch.equal(exponent, want[1])
    with pytest.raises(ValueError, match="exponent per 32 dims"):
        copy_kv_blocks(payload.view(FP4), [(0, 3)], exponent.view(E8M0)[..., 0])


# ---- refusals


def caches(dim=128, page=16, heads=2):
    (kc, ks), (vc, vs) = (empty_cache((4, page, heads, dim), device="cpu") for _ in range(2))
    return dict(k_cache=kc, v_cache=vc, k_scale_cache=ks, v_scale_cache=vs)


SCALE_REFUSALS = [
    (lambda c: c.update(k_scale_cache=None, v_scale_cache=None), "need their exponents"),
    (lambda c: c.update(k_scale_cache=c["k_scale_cache"][..., :2]), "exponent"),
    (lambda c: c.update(v_scale_cache=torch.ones(4, 16, 2)), "exponent|scale"),
    (lambda c: c.update({n: c[n].view(torch.uint8) for n in ("k_scale_cache", "v_scale_cache")}), "float8_e8m0fnu"),
]


@pytest.mark.parametrize("change,match", SCALE_REFUSALS)
@pytest.mark.parametrize("op", ["store", "rotate", "load", "decode", "prefill"])
def test_exponents_that_do_not_fit(op, change, match):
    c = caches()
    change(c)
    with pytest.raises(ValueError, match=match):
        call(op, c)


def call(op, c, **kw):
    tokens = 3
    x = dict(q=torch.zeros(tokens, 4, 128, dtype=BF16), key=torch.zeros(tokens, 2, 128, dtype=BF16),
             value=torch.zeros(tokens, 2, 128, dtype=BF16), cos_sin=torch.zeros(9, 128),
             positions=torch.zeros(tokens, dtype=torch.int32), slot_mapping=torch.arange(tokens, dtype=torch.int32),
             block_tables=torch.zeros(tokens, 2, dtype=torch.int32), context_lens=torch.ones(tokens, dtype=torch.int32),
             cu_seqlens_q=torch.tensor([0, 1, 2, 3], dtype=torch.int32), max_context_len=torch.tensor(1, dtype=torch.int32),
             position_axes=None, num_heads=4, num_kv_heads=2, dtype=BF16, block_n=16) | kw
    scales = dict(k_scale_cache=c["k_scale_cache"], v_scale_cache=c["v_scale_cache"])
    if op == "store":
        return store_kvcache(x["key"], x["value"], c["k_cache"], c["v_cache"], x["slot_mapping"], **scales)
    if op == "rotate":
        return rotate_store_kvcache(x["q"], x["key"], x["value"], x["cos_sin"], x["positions"], c["k_cache"], c["v_cache"],
                                    x["slot_mapping"], position_axes=x["position_axes"], **scales)
    if op == "load":
        return load_kvcache(c["k_cache"], c["v_cache"], x["slot_mapping"], dtype=x["dtype"], **scales)
    if op == "decode":
        return paged_decode_attention(x["q"], c["k_cache"], c["v_cache"], x["block_tables"], x["context_lens"], 0.1,
                                      max_context_len=x["max_context_len"], block_n=x["block_n"], **scales)
    context = SimpleNamespace(block_tables=x["block_tables"], context_lens=x["context_lens"], cu_seqlens_q=x["cu_seqlens_q"])
    return paged_prefill_attention(x["q"], c["k_cache"], c["v_cache"], context, num_heads=x["num_heads"], num_kv_heads=x["num_kv_heads"],
                                   scale=0.1, **scales)


REFUSALS = [
    # rotation
    ("rotate", dict(q=torch.zeros(2, 4, 128, dtype=BF16)), ValueError, "q must be"),
    ("rotate", dict(q=torch.zeros(3, 4, 64, dtype=BF16)), ValueError, "q must be"),
    ("rotate", dict(cos_sin=torch.zeros(9, 65)), ValueError, "cos_sin must be"),
    ("rotate", dict(cos_sin=torch.zeros(9, 130)), ValueError, "cos_sin must be"),
    ("rotate", dict(cos_sin=torch.zeros(9, 0)), ValueError, "cos_sin must be"),
    ("rotate", dict(cos_sin=torch.zeros(9, 128, dtype=BF16)), ValueError, "cos_sin must use torch.float32"),
    ("rotate", dict(positions=torch.zeros(3, dtype=torch.long)), ValueError, "positions must use torch.int32"),
    ("rotate", dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions must be"),
    ("rotate", dict(positions=torch.zeros(3, 3, dtype=torch.int32)), ValueError, "without position_axes"),
    ("rotate", dict(position_axes=torch.zeros(64, dtype=torch.int32)), ValueError, "with position_axes"),
    ("rotate", dict(positions=torch.zeros(3, 3, dtype=torch.int32), position_axes=torch.zeros(63, dtype=torch.int32)), ValueError, "position_axes must be"),
    ("rotate", dict(positions=torch.zeros(3, 3, dtype=torch.int32), position_axes=torch.zeros(64)), ValueError, "position_axes must be"),
    ("rotate", dict(q=torch.zeros(3, 4, 128)), ValueError, "one dtype"),
    ("rotate", dict(value=torch.zeros(3, 2, 64, dtype=BF16)), ValueError, "same"),
    ("rotate", dict(key=torch.zeros(3, 3, 128, dtype=BF16), value=torch.zeros(3, 3, 128, dtype=BF16)), ValueError, "head shape mismatch"),
    ("rotate", dict(slot_mapping=torch.zeros(2, dtype=torch.int32)), ValueError, "one flat slot per input token"),
    ("rotate", {}, RuntimeError, "runs on the GPU"),
    # reading back
    ("load", dict(dtype=torch.float64), ValueError, "dtype must be"),
    ("load", dict(slot_mapping=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "one flat slot"),
    ("load", {}, RuntimeError, "runs on the GPU"),
    # attention
    ("decode", dict(q=torch.zeros(3, 4, 64, dtype=BF16)), ValueError, "head_dim mismatch"),
    ("decode", dict(q=torch.zeros(3, 3, 128, dtype=BF16)), ValueError, "divisible"),
    ("decode", dict(q=torch.zeros(3, 128, dtype=BF16)), ValueError, "q must be"),
    ("decode", dict(q=torch.zeros(3, 4, 128)), RuntimeError, "bf16 or float16 queries"),
    ("decode", dict(block_n=12), ValueError, "power of two"),
    ("decode", dict(block_tables=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "must cover q batch"),
    ("decode", {}, RuntimeError, "no CPU fallback"),
    ("prefill", dict(num_heads=6, num_kv_heads=2), ValueError, "q must be"),
    ("prefill", dict(num_kv_heads=4), ValueError, "num_kv_heads=4"),
    ("prefill", dict(num_kv_heads=3), ValueError, "divisible"),
    ("prefill", dict(q=torch.zeros(3, 4, 64, dtype=BF16)), ValueError, "head_dim mismatch"),
    ("prefill", dict(q=torch.zeros(3, 4, 128)), RuntimeError, "bf16 or float16 queries"),
    ("prefill", dict(block_tables=torch.zeros(4, dtype=torch.int32)), ValueError, "two-dimensional"),
    ("prefill", dict(block_tables=None), RuntimeError, "requires block_tables"),
    ("prefill", {}, RuntimeError, "no CPU fallback"),
    # the store
    ("store", dict(key=torch.zeros(3, 2, 64, dtype=BF16), value=torch.zeros(3, 2, 64, dtype=BF16)), ValueError, "head shape mismatch"),
]


@pytest.mark.parametrize("op,change,error,match", REFUSALS, ids=lambda x: x if isinstance(x, str) else None)
def test_calls_that_are_refused(op, change, error, match):
    with pytest.raises(error, match=match):
        call(op, caches(), **change)


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_geometries_that_are_refused(op):
    with pytest.raises(RuntimeError, match="multiple of 16 tokens"):
        call(op, caches(page=8))
    with pytest.raises(RuntimeError, match="head_dim 64 and 128"):
        call(op, caches(dim=96), q=torch.zeros(3, 4, 96, dtype=BF16))
    q = torch.zeros(3, 4, 128, dtype=BF16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(op, caches(), q=q)
    mixed = caches()
    mixed["v_cache"] = mixed["v_cache"].view(FP8)
    with pytest.raises(ValueError):
        call(op, mixed)


# ---- the C entries: error codes, never a launch


@pytest.fixture
def native():
    from prism_infer import _native

    if not _native.available():
        pytest.skip("the library is not built")
    return _native.lib(), _native.int64s


P = 4096  # an address that nothing reads


def rotate(lib, int64s, **kw):
    a = dict(q=P, key=P, value=P, in_dtype=1, cos_sin=P, max_positions=9, rotary=128, pairs=0, positions=P, stride=3, num_axes=1, axes=None,
             q_out=P, key_out=None, k_cache=P, v_cache=P, cache=4, ks=P, vs=P, slots=P, tokens=3, heads=4, kv_heads=2, dim=128, num_slots=64,
             strides=int64s(512, 128, 1)) | kw
    s = a.pop("strides")
    rc = lib.prism_kv_rotate_store(a["q"], s, a["key"], s, a["value"], s, a["in_dtype"], a["cos_sin"], a["max_positions"], a["rotary"],
                                   a["pairs"], a["positions"], a["stride"], a["num_axes"], a["axes"], a["q_out"], a["key_out"], a["k_cache"],
                                   a["v_cache"], a["cache"], a["ks"], a["vs"], a["slots"], a["tokens"], a["heads"], a["kv_heads"], a["dim"],
                                   a["num_slots"], None)
    return rc, lib.prism_last_error().decode()


@pytest.mark.parametrize("change,match", [(dict([(n, None)]), "null") for n in ("q", "key", "value", "cos_sin", "positions", "q_out", "k_cache", "v_cache", "slots")]
                         + [(dict(ks=None), ""), (dict(ks=None, vs=None), ""), (dict(in_dtype=3), "input dtype"), (dict(in_dtype=4), "input dtype"),
                            (dict(cache=9), ""), (dict(rotary=127), "rotary_dim"), (dict(rotary=130), "rotary_dim"), (dict(num_axes=0), "rotary_dim"),
                            (dict(dim=80, rotary=64), ""), (dict(tokens=-1), "geometry"), (dict(kv_heads=0), "geometry"), (dict(num_slots=-1), "geometry"),
                            (dict(tokens=2 ** 31), "geometry"), (dict(tokens=2 ** 29), "too many rows"), (dict(heads=2 ** 31 - 1), "too many rows")])
def test_the_rotation_entrys_errors(native, change, match):
    rc, message = rotate(*native, **change)
    assert rc < 0 and message.startswith("prism_kv_rotate_store") and match in message, (rc, message)


def test_the_rotation_entry_needs_unit_strides(native):
    rc, message = rotate(*native, strides=native[1](512, 128, 2))
    assert rc < 0 and "unit-stride" in message


def test_entries_without_rows_read_nothing(native):
    names = ("q", "key", "value", "cos_sin", "positions", "q_out", "k_cache", "v_cache", "slots")
    assert rotate(*native, tokens=0, **dict.fromkeys(names))[0] == 0
    lib = native[0]
    assert lib.prism_kv_load(None, None, 1, None, None, None, None, None, 1, 0, 2, 128, 4, None) == 0
    assert attention(*native, batch=0, **dict.fromkeys(("q", "k", "v", "bt", "ctx", "out")))[0] == 0


@pytest.mark.parametrize("args,match", [((P, P, 4, P, None, P, P, P, 1, 3, 2, 128, 64), ""), ((P, P, 1, None, None, None, P, P, 1, 3, 2, 128, 64), "null"),
                                        ((None, P, 1, None, None, P, P, P, 1, 3, 2, 128, 64), "null"), ((P, P, 1, None, None, P, P, P, 3, 3, 2, 128, 64), "output dtype"),
                                        ((P, P, 1, None, None, P, P, P, 1, 3, 2, 12, 64), "multiple of 8"), ((P + 8, P, 1, None, None, P, P, P, 1, 3, 2, 128, 64), "aligned"),
                                        ((P, P, 1, None, None, P, P, P, 1, 3, 0, 128, 64), "geometry"), ((P, P, 1, None, None, P, P, P, 1, 2 ** 28, 2, 128, 64), "too many")])
def test_the_load_entrys_errors(native, args, match):
    lib = native[0]
    rc = lib.prism_kv_load(*args, None)
    message = lib.prism_last_error().decode()
    assert rc < 0 and message.startswith("prism_kv_load") and match in message, (rc, message)


def attention(lib, int64s, **kw):
    a = dict(q=P, q_dtype=1, k=P, v=P, ke=P, ve=P, bt=P, ctx=P, max_ctx=P, cu=None, out=P, batch=2, total=2, heads=4, kv_heads=2, dim=128, page=16,
             blocks=8, width=4, status=None, ws=P, short=0, qs=int64s(512, 128, 1), ks=int64s(2048, 128, 64, 1), es=int64s(128, 8, 4, 1)) | kw
    need = lib.prism_paged_fp4_workspace_bytes(int(a["cu"] is not None), a["batch"], a["total"], a["heads"], a["kv_heads"], a["dim"], a["page"], a["width"])
    rc = lib.prism_paged_fp4(a["q"], a["q_dtype"], a["qs"], a["k"], a["v"], a["ks"], a["ks"], a["ke"], a["ve"], a["es"], a["es"], a["bt"],
                             int64s(4, 1), a["ctx"], a["max_ctx"], a["cu"], a["out"], a["qs"], a["batch"], a["total"], a["heads"], a["kv_heads"],
                             a["dim"], a["page"], a["blocks"], a["width"], 0.1, a["status"], None, a["ws"], need - a["short"], None)
    return rc, lib.prism_last_error().decode()


@pytest.mark.parametrize("change,match", [(dict([(n, None)]), "null") for n in ("q", "k", "v", "ke", "ve", "bt", "ctx", "max_ctx", "out")]
                         + [(dict(cu=P), "null"), (dict(q_dtype=0), "bf16 or float16"), (dict(q_dtype=4), "bf16 or float16"), (dict(dim=96), "head_dim"),
                            (dict(page=24), "multiple of 16"), (dict(page=0), "geometry"), (dict(kv_heads=3), "geometry"), (dict(width=-1), "geometry"),
                            (dict(total=1), "query rows"), (dict(q=P + 2), "aligned"), (dict(k=P + 8), "aligned"), (dict(ke=P + 1), "aligned"),
                            (dict(short=1), "workspace"), (dict(ws=None), "workspace"), (dict(ws=P + 128), "workspace"),
                            (dict(width=2 ** 31 - 1, batch=4096, total=4096), "too many steps")])
def test_the_attention_entrys_errors(native, change, match):
    rc, message = attention(*native, **change)
    assert rc < 0 and message.startswith("prism_paged_fp4") and match in message, (rc, message)


def test_the_attention_entrys_strides(native):
    int64s = native[1]
    for change in (dict(qs=int64s(512, 128, 2)), dict(qs=int64s(516, 128, 1)), dict(ks=int64s(2048, 128, 64, 2)), dict(ks=int64s(2048, 72, 64, 1)),
                   dict(es=int64s(128, 8, 2, 1)), dict(ks=int64s(2 ** 40, 2 ** 27, 64, 1)), dict(ks=int64s(2 ** 40, 128, 2 ** 29, 1))):
        rc, message = attention(*native, **change)
        assert rc < 0 and message.startswith("prism_paged_fp4"), (rc, message)
