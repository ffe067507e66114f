"""Rotation, 4-bit stores, reads and attention through the native host path and through Python: the same results and errors."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _fp4 import Pool, attend, check
from _helpers import require_gpu
from prism_infer import observability
from prism_infer.ops import kv_cache_load, kv_cache_store, paged_decode, paged_prefill, rotary_kv_store
from test_gpu_rotary_store import make, make_cache, same_bytes, table

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
MODULES = (kv_cache_load, kv_cache_store, paged_decode, paged_prefill, rotary_kv_store)


def python(monkeypatch, call):
    with monkeypatch.context() as m:
        for module in MODULES:
            m.setattr(module, "_HOST", None)
        return call()


def expect_native(monkeypatch, name):
    """Make the op's native call fail the test where it declines."""

    class Host:
        def __getattr__(self, attr):
            real = getattr(kv_cache_load._native.host_ops(), attr)

            def wrapped(*args):
                out = real(*args)
                assert attr != name or out not in (None, False), f"{name} was left to Python"
                return out

            return wrapped

    for module in MODULES:
        monkeypatch.setattr(module, "_HOST", Host())


@pytest.mark.parametrize("kind", ["fp4", "fp8", "fp8_unit", "bf16"])
@pytest.mark.parametrize("axes", [1, 3])
def test_rotation_store_and_load(monkeypatch, kind, axes):
    require_gpu()
    q, k, v, g = make(33, 8, 2, 128, BF16, seed=1)
    cos_sin = table(64, 128).cuda()
    positions = torch.randint(0, 64, (axes, 33), generator=g, dtype=torch.int32).cuda()
    which = torch.randint(0, axes, (64,), generator=g, dtype=torch.int32).cuda() if axes > 1 else None
    slots = torch.randperm(64, generator=g)[:33].int().cuda()
    caches = [make_cache(kind, 4, 16, 2, 128) for _ in range(4)]

    def rotate(c):
        return rotary_kv_store.rotate_store_kvcache(q, k, v, cos_sin, positions if axes > 1 else positions[0], *c[:2], slots, *c[2:],
                                                    position_axes=which, return_key=True)

    def store(c):
        kv_cache_store.store_kvcache(k, v, *c[:2], slots, *c[2:])

    def load(c):
        return kv_cache_load.load_kvcache(*c[:2], slots, *c[2:], dtype=torch.float32)

    got = python(monkeypatch, lambda: (rotate(caches[0]), load(caches[0])))
    python(monkeypatch, lambda: store(caches[1]))
    for name in ("rotate_store", "load", "store"):
        expect_native(monkeypatch, name)
    want = rotate(caches[2]), load(caches[2])
    store(caches[3])
    for a, b in zip((*got[0], *got[1]), (*want[0], *want[1])):
        assert same_bytes(a, b)
    for one, two in ((0, 2), (1, 3)):
        assert all(same_bytes(a, b) for a, b in zip(caches[one], caches[two]) if a is not None)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention(monkeypatch, dtype):
    require_gpu()
    pool = Pool([300, 0, 41], page=16, kv_heads=2, dim=128, seed=3)
    g = torch.Generator().manual_seed(4)
    one, chunk = (torch.randn(n, 8, 128, generator=g).to(dtype).cuda() for n in (3, 60))
    context = SimpleNamespace(block_tables=pool.tables[[0, 2]], context_lens=pool.lens[[0, 2]],
                              cu_seqlens_q=torch.tensor([0, 37, 60], dtype=torch.int32, device="cuda"))
    scales = dict(k_scale_cache=pool.ks, v_scale_cache=pool.vs)
    decode = lambda: paged_decode.paged_decode_attention(one, pool.kc, pool.vc, pool.tables, pool.lens, 0.09, **scales)  # noqa: E731
    prefill = lambda c=context: paged_prefill.paged_prefill_attention(chunk, pool.kc, pool.vc, c, num_heads=8, num_kv_heads=2,  # noqa: E731
                                                                      scale=0.09, **scales)
    want = python(monkeypatch, decode), python(monkeypatch, prefill)
    wide = SimpleNamespace(**{n: t.long() for n, t in vars(context).items()})  # int64, which Python converts
    assert torch.equal(prefill(wide), want[1])
    for name in ("decode", "prefill"):
        expect_native(monkeypatch, name)
    assert torch.equal(decode(), want[0]) and torch.equal(prefill(), want[1])


def test_errors_are_the_same(monkeypatch):
    require_gpu()
    pool = Pool([40, 20], page=16, kv_heads=2, dim=128, seed=5)
    q = torch.randn(30, 8, 128, device="cuda").to(BF16)
    k = torch.randn(30, 2, 128, device="cuda").to(BF16)
    slots, cos_sin = torch.arange(30, dtype=torch.int32, device="cuda"), table(64, 128).cuda()
    scales = dict(k_scale_cache=pool.ks, v_scale_cache=pool.vs)

    def prefill(lens=(40, 20), cu=(0, 20, 30), tables=pool.tables):
        context = SimpleNamespace(block_tables=tables, context_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                  cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        return paged_prefill.paged_prefill_attention(q, pool.kc, pool.vc, context, num_heads=8, num_kv_heads=2, scale=0.1, **scales)

    def rotate(**kw):
        a = dict(q=q, key=k, value=k, cos_sin=cos_sin, positions=slots, k_cache=pool.kc, v_cache=pool.vc, slot_mapping=slots, **scales) | kw
        return rotary_kv_store.rotate_store_kvcache(**a)

    bad = pool.tables.clone()
    bad[1, 0] = pool.kc.shape[0]
    calls = [
        lambda: prefill(lens=(15, 20)), lambda: prefill(cu=(0, 30, 30)), lambda: prefill(lens=(40, 80)), lambda: prefill(tables=bad),
        lambda: rotate(positions=slots.long()), lambda: rotate(slot_mapping=slots.long()), lambda: rotate(cos_sin=cos_sin[:, :127]),
        lambda: rotate(key=k.float()), lambda: rotate(k_scale_cache=None), lambda: rotate(k_cache=pool.kc[:, :8]),
        lambda: rotate(q=q.clone().requires_grad_()), lambda: rotate(cos_sin=cos_sin.cpu()), lambda: rotate(k_cache=pool.kc.transpose(1, 2)),
        lambda: rotate(q=q.transpose(1, 2)), lambda: rotate(value=k.transpose(0, 1)),
        lambda: kv_cache_load.load_kvcache(pool.kc, pool.vc, slots.long(), **scales),
        lambda: kv_cache_load.load_kvcache(pool.kc, pool.vc, slots[::2], **scales),
        lambda: kv_cache_store.store_kvcache(k.double(), k.double(), pool.kc, pool.vc, slots, pool.ks, pool.vs),
        lambda: paged_decode.paged_decode_attention(q.cpu(), pool.kc, pool.vc, pool.tables, pool.lens, 0.1, **scales),
        lambda: paged_decode.paged_decode_attention(q[:2], pool.kc, pool.vc, pool.tables, pool.lens, 0.1),
    ]
    before = [t.clone() for t in (pool.kc, pool.vc, pool.ks, pool.vs)]
    for i, call in enumerate(calls):
        with pytest.raises((ValueError, RuntimeError)) as native:
            call()
        with pytest.raises(type(native.value)) as plain:
            python(monkeypatch, call)
        assert str(native.value) == str(plain.value), i
    assert all(same_bytes(a, b) for a, b in zip(before, (pool.kc, pool.vc, pool.ks, pool.vs)))


def test_tensors_that_the_native_path_leaves(monkeypatch):
    """Strided slots, positions and angles, and exponents off their length: taken all the same, with the same results."""

    require_gpu()
    q, k, v, g = make(20, 8, 2, 128, BF16, seed=6)
    cos_sin, slots = table(64, 128).cuda(), torch.randperm(64, generator=g)[:20].int().cuda()
    positions = torch.arange(20, dtype=torch.int32, device="cuda")
    spread = lambda t: torch.stack([t, t], -1)[..., 0]  # noqa: E731  (the same values, strided)
    one, two = make_cache("fp4", 4, 16, 2, 128), make_cache("fp4", 4, 16, 2, 128)
    off = [torch.empty(c.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(c.shape) for c in one[2:]]
    for o, c in zip(off, one[2:]):
        o.copy_(c.view(torch.uint8))
    off = [o.view(torch.float8_e8m0fnu) for o in off]
    want = rotary_kv_store.rotate_store_kvcache(q, k, v, cos_sin, positions, *two[:2], slots, *two[2:])
    got = rotary_kv_store.rotate_store_kvcache(q, k, v, spread(cos_sin), spread(positions), *one[:2], spread(slots), *off)
    assert same_bytes(got, want) and all(same_bytes(a, b) for a, b in zip((*one[:2], *off), two))
    tables, lens = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device="cuda"), torch.tensor([64], dtype=torch.int32, device="cuda")
    a = paged_decode.paged_decode_attention(q[:1], *one[:2], tables, lens, 0.1, k_scale_cache=off[0], v_scale_cache=off[1])
    b = paged_decode.paged_decode_attention(q[:1], *two[:2], tables, lens, 0.1, k_scale_cache=two[2], v_scale_cache=two[3])
    assert torch.equal(a, b)
    loaded = kv_cache_load.load_kvcache(*one[:2], slots, *off), kv_cache_load.load_kvcache(*two[:2], slots, *two[2:])
    assert all(same_bytes(x, y) for x, y in zip(*loaded))


def test_profile_regions():
    require_gpu()
    seen = []

    class Region:
        def __init__(self, name, **kwargs):
            seen.append((name, kwargs["metadata"]["tokens"]))

        def __enter__(self):
            return self

        def __exit__(self, *exc):
            return False

    q, k, v, _ = make(5, 8, 2, 128, BF16, seed=7)
    cos_sin, slots = table(64, 128).cuda(), torch.arange(5, dtype=torch.int32, device="cuda")
    observability.install_performance_provider(profile_region_provider=Region, profile_session_provider=lambda: None)
    try:
        for kind in ("fp4", "fp8", "bf16"):
            c = make_cache(kind, 4, 16, 2, 128)
            rotary_kv_store.rotate_store_kvcache(q, k, v, cos_sin, slots, *c[:2], slots, *c[2:])
        c = make_cache("fp4", 4, 16, 2, 128)
        kv_cache_store.store_kvcache(k, v, *c[:2], slots, *c[2:])
    finally:
        observability._reset_performance_providers()
    assert seen == [(f"attention.kv_store.hip{x}", 5) for x in ("_fp4", "_scaled_fp8", "", "_fp4")]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [4, 8])
def test_a_bad_query_spoils_its_own_rows_only(dtype, group):
    """NaN and infinite queries beside good ones of the same block of rows."""

    require_gpu()
    pool = Pool([700, 150, 64], page=16, kv_heads=2, dim=128, seed=8)
    g = torch.Generator().manual_seed(9)
    heads = 2 * group
    q = torch.randn(3, heads, 128, generator=g).to(dtype)
    q[0, 1, 5], q[0, heads - 1, 100], q[1, 2, 0] = torch.nan, torch.inf, -torch.inf
    bad = {(0, 1), (0, heads - 1), (1, 2)}
    scales = dict(k_scale_cache=pool.ks, v_scale_cache=pool.vs)
    got = paged_decode.paged_decode_attention(q.cuda(), pool.kc, pool.vc, pool.tables, pool.lens, 0.09, **scales).cpu()
    context = SimpleNamespace(block_tables=pool.tables, context_lens=pool.lens, cu_seqlens_q=torch.arange(4, dtype=torch.int32, device="cuda"))
    chunk = paged_prefill.paged_prefill_attention(q.cuda(), pool.kc, pool.vc, context, num_heads=heads, num_kv_heads=2, scale=0.09, **scales).cpu()
    for i in range(3):
        k, v, keep = pool.rows(i)
        seen = torch.ones(1, keep.numel(), dtype=torch.bool)
        for h in range(heads):
            if (i, h) in bad:
                assert not got[i, h].isfinite().any() and not chunk[i, h].isfinite().any(), (i, h)
                continue
            for out, weight in ((got, 2.0 ** -8 if dtype == BF16 else 2.0 ** -16), (chunk, 2.0 ** -8 if dtype == BF16 else 2.0 ** -11)):
                want, bound = attend(q[i, h][None].double(), k[:, h // group], v[:, h // group], 0.09, seen, weight)
                check(out[i, h][None], want, bound, f"{i}, {h}")


@pytest.mark.parametrize("kind", ["fp4", "fp8", "bf16"])
def test_flat_caches_and_slots_named_twice(monkeypatch, kind):
    """[slots, heads, dim] caches are the paged ones' rows; a slot may be read back any number of times."""

    require_gpu()
    q, k, v, g = make(24, 8, 2, 128, BF16, seed=10)
    cos_sin, slots = table(64, 128).cuda(), torch.randperm(64, generator=g)[:24].int().cuda()
    positions = torch.arange(24, dtype=torch.int32, device="cuda")
    paged = make_cache(kind, 4, 16, 2, 128)
    flat = [None if c is None else c.clone().flatten(0, 1) for c in paged]
    want = rotary_kv_store.rotate_store_kvcache(q, k, v, cos_sin, positions, *paged[:2], slots, *paged[2:])
    twice = torch.cat([slots, slots.flip(0), torch.tensor([-1, 64, 2 ** 31 - 1], dtype=torch.int32, device="cuda")])
    for native in (True, False):
        call = lambda: (rotary_kv_store.rotate_store_kvcache(q, k, v, cos_sin, positions, *flat[:2], slots, *flat[2:]),  # noqa: E731
                        kv_cache_load.load_kvcache(*flat[:2], twice, *flat[2:]))
        got, (key, value) = call() if native else python(monkeypatch, call)
        assert same_bytes(got, want) and all(same_bytes(a.flatten(0, 1), b) for a, b in zip(paged, flat) if a is not None)
        for rows in (key, value):
            assert same_bytes(rows[:24], rows[24:48].flip(0)) and bool((rows[48:] == 0).all())
