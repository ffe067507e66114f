"""Layers with a bound rotation over every kind of cache: prompts, chunks, decode steps, moved blocks, one graph.

What the layers rotate and store is defined to the last bit (test_gpu_rotary_store), so the pages are compared bytes for
bytes with the tokens so far, rotated on the host; attention is compared with plain attention in 64 bits over what the
pages hold (over the rotated keys themselves where a prompt has nothing in front of it).
"""

from __future__ import annotations

import math

import pytest
import torch

from _attention16 import assert_within, attention64
from _fp4 import E8M0, FP4, attend, check, decode, empty_cache
from _helpers import require_gpu
from test_gpu_rotary_store import make_cache, rotated, same_bytes, stored, table
from test_gpu_serving_steps import Requests

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
KINDS = {"16bit": {BF16: "bf16", F16: "f16"}, "scaled": {BF16: "fp8"}, "4bit": {BF16: "fp4", F16: "fp4"}}


class RotaryRequests(Requests):
    """Requests whose layers rotate; their tokens so far are kept rotated."""

    def __init__(self, batch, heads, kv_heads, dtype, cache, *, rotary=128, pairs=False, axes=None, **kwargs):
        super().__init__(batch, heads, kv_heads, dtype, "16bit", **kwargs)
        self.kind, self.pairs, self.axes = KINDS[cache][dtype], pairs, axes
        self.caches = make_cache(self.kind, self.free.numel(), self.page, kv_heads, 128)
        self.table = table(700, rotary)
        for layer in (self.prefill, self.decode):
            layer.k_cache, layer.v_cache, layer.k_scale_cache, layer.v_scale_cache = self.caches
            layer.cos_sin_cache, layer.interleaved_rotary = self.table.cuda(), pairs
            layer.position_axes = None if axes is None else axes.cuda()

    def tokens(self, new, rows, positions=None):
        """(q, k, v as views of one packed projection, q rotated); k rotated and v are remembered."""

        h, g = self.heads, self.kv_heads
        qkv = torch.randn(rows, (h + 2 * g) * 128, generator=self.g).to(self.dtype)
        if positions is None:
            at = [torch.arange(len(k), len(k) + n) for k, n in zip(self.k, new)]
            positions = torch.cat([*at, torch.zeros(rows - sum(new), dtype=torch.long)]).int()
        split = lambda x: [t.unflatten(1, (-1, 128)) for t in x.split([h * 128, g * 128, g * 128], 1)]  # noqa: E731
        q, k, v = split(qkv)
        q, k = (rotated(x, self.table, positions, self.axes, self.pairs) for x in (q, k))
        at = 0
        for i, n in enumerate(new):
            self.k[i], self.v[i] = torch.cat([self.k[i], k[at:at + n]]), torch.cat([self.v[i], v[at:at + n]])
            at += n
        return split(qkv.cuda()), q

    def stored(self, i):
        """Request i's tokens as its pages hold them, in 64 bits; their bytes are those of the definition."""

        n = self.k[i].shape[0]
        pages = self.tables[i, :-(-n // self.page)].long()
        rows = []
        for payload, scales, tokens in ((self.caches[0], self.caches[2], self.k[i]), (self.caches[1], self.caches[3], self.v[i])):
            pick = lambda c: c.view(torch.uint8)[pages].flatten(0, 1)[:n].cpu().contiguous().view(c.dtype)  # noqa: E731
            got, want = (pick(payload), None if scales is None else pick(scales)), stored(tokens, self.kind, payload.dtype)
            if n:
                assert same_bytes(got[0], want[0]) and (want[1] is None or same_bytes(got[1], want[1])), f"request {i}"
            if self.kind == "fp4":
                rows.append(decode(*got) if n else torch.zeros(0, self.kv_heads, 128, dtype=torch.float64))
            else:
                rows.append(got[0].double() * (1.0 if got[1] is None else got[1].double()[..., None]))
        return rows

    def compare(self, q, got, new, *, own_keys, step=False):
        at = 0
        for i, n in enumerate(new):
            k, v = self.stored(i)
            if n == 0:
                continue
            rows, label = slice(at, at + n), f"request {i}"
            if own_keys or self.kind != "fp4":
                k, v = (self.k[i], self.v[i]) if own_keys else (k, v)
                want, bound = attention64(q[rows], k, v, self.scale)
                # the step's op over 16-bit and FP8 caches has the reference's bound, as chunks over FP8 have
                loose = not own_keys and (step or self.kind == "fp8")
                assert_within(got[rows], want, torch.full_like(bound, 2e-2) if loose else bound, label)
            else:
                weight = 2.0 ** -8 if self.dtype == BF16 else 2.0 ** -16 if step else 2.0 ** -11
                group, m = self.heads // self.kv_heads, k.shape[0]
                seen = torch.arange(m)[None, :] <= (m - n + torch.arange(n))[:, None]
                for h in range(self.heads):
                    want, bound = attend(q[rows, h].double(), k[:, h // group], v[:, h // group], self.scale, seen, weight)
                    check(got[rows, h], want, bound, f"{label}, head {h}")
            at += n


@pytest.mark.parametrize("cache,dtype,rotary,pairs", [("16bit", BF16, 128, False), ("16bit", F16, 64, True), ("scaled", BF16, 128, False),
                                                      ("4bit", BF16, 128, False), ("4bit", F16, 128, True)])
def test_prompts_chunks_and_decode_steps(cache, dtype, rotary, pairs):
    require_gpu()
    r = RotaryRequests(5, 8, 2, dtype, cache, rotary=rotary, pairs=pairs)
    new = [37, 1, 64, 90, 17]  # prompts, padded to 256 rows
    m = r.metadata(new, 256)
    (q, k, v), turned = r.tokens(new, 256)
    out = r.prefill(q, k, v, m, cached_prefix=False)
    r.compare(turned, out, new, own_keys=True)
    assert (out[sum(new):] == 0).all()
    new = [100, 3, 64, 1, 45]  # a chunk behind each of them
    m = r.metadata(new, sum(new))
    (q, k, v), turned = r.tokens(new, sum(new))
    r.compare(turned, r.prefill(q, k, v, m, cached_prefix=True), new, own_keys=False)
    for _ in range(12):
        new = [1] * r.batch
        m = r.metadata(new, r.batch)
        (q, k, v), turned = r.tokens(new, r.batch)
        out = r.decode(q, k, v, _as_decode(m), m.positions)
        r.compare(turned, out, new, own_keys=False, step=True)


def _as_decode(m):
    """The step's metadata as a decode step packs it, which has no positions."""

    from prism_infer.engine.decode_attention import pack_decode_metadata

    packed = pack_decode_metadata(m.slot_mapping.tolist(), m.context_lens.tolist(), m.block_tables, device="cuda")
    assert getattr(packed, "positions", None) is None
    return packed


@pytest.mark.parametrize("cache", ["4bit", "scaled"])
def test_positions_of_several_axes(cache):
    """Text, height and width positions by section, given with the call."""

    require_gpu()
    axes = torch.tensor([0] * 24 + [1] * 20 + [2] * 20, dtype=torch.int32)
    r = RotaryRequests(2, 4, 2, BF16, cache, axes=axes)
    new = [40, 9]
    m = r.metadata(new, sum(new))
    positions = torch.randint(0, 600, (3, sum(new)), generator=r.g, dtype=torch.int32)
    (q, k, v), turned = r.tokens(new, sum(new), positions)
    out = r.prefill(q, k, v, m, positions.cuda(), cached_prefix=False)
    r.compare(turned, out, new, own_keys=True)
    m = r.metadata([1, 1], 2)
    positions = torch.randint(0, 600, (3, 2), generator=r.g, dtype=torch.int32)
    (q, k, v), turned = r.tokens([1, 1], 2, positions)
    r.compare(turned, r.decode(q, k, v, m, positions.cuda()), [1, 1], own_keys=False, step=True)


def test_blocks_of_a_4bit_cache_move_with_their_exponents():
    """Copy-on-write, a prefix's rows, compacted slots, and blocks out to the host and back: the same bytes, so the same output."""

    require_gpu()
    from prism_infer.engine.kv_block_ops import copy_kv_block_prefixes, copy_kv_blocks, swap_blocks
    from prism_infer.ops.kv_compaction import compact_kv_slots
    from prism_infer.ops.paged_decode import paged_decode_attention

    g = torch.Generator().manual_seed(5)
    payload = torch.randint(0, 256, (2, 3, 12, 16, 2, 64), generator=g, dtype=torch.uint8).cuda()
    exponent = torch.randint(120, 132, (2, 3, 12, 16, 2, 4), generator=g, dtype=torch.uint8).cuda()
    kv, scales = payload.view(FP4), exponent.view(E8M0)
    q = torch.randn(1, 8, 128, generator=g).to(BF16).cuda()

    def attended(blocks, n, layer=1):
        return paged_decode_attention(q, kv[0, layer], kv[1, layer], torch.tensor([blocks], dtype=torch.int32, device="cuda"),
                                      torch.tensor([n], dtype=torch.int32, device="cuda"), 0.09, k_scale_cache=scales[0, layer],
                                      v_scale_cache=scales[1, layer])

    want = attended([3, 7, 2], 40)
    copy_kv_blocks(kv, [(3, 0), (7, 1)], scales)
    copy_kv_block_prefixes(kv, [(2, 5, 8)], scales)
    assert torch.equal(attended([0, 1, 5], 40), want)
    assert torch.equal(payload[:, :, 5, :8], payload[:, :, 2, :8]) and torch.equal(exponent[:, :, 5, :8], exponent[:, :, 2, :8])
    host = torch.zeros((2, 3, 4, 16, 2, 64), dtype=torch.uint8).pin_memory(), torch.zeros((2, 3, 4, 16, 2, 4), dtype=torch.uint8).pin_memory()
    ids = dict(gpu_scale_cache=scales, cpu_scale_cache=host[1].view(E8M0))
    swap_blocks(kv, host[0].view(FP4), [(0, 3), (1, 1), (5, 0)], "out", **ids)
    payload[:, :, [0, 1, 5]], exponent[:, :, [0, 1, 5]] = 0, 255
    assert attended([0, 1, 5], 40).isnan().all()
    swap_blocks(kv, host[0].view(FP4), [(3, 8), (1, 9), (0, 10)], "in", **ids)
    assert torch.equal(attended([8, 9, 10], 40), want)
    # the sequence's tokens to the front of blocks 0 to 2
    src = torch.cat([torch.arange(b * 16, b * 16 + 16) for b in (8, 9, 10)])[:40].cuda()
    dst = torch.arange(40).cuda()
    for cache in (kv, scales):
        compact_kv_slots(cache.view(2, 3, 192, 2, -1), src, dst)
    assert torch.equal(attended([0, 1, 2], 40), want)
    with pytest.raises(ValueError, match="exponent per 32 dims"):
        copy_kv_blocks(kv, [(0, 1)], scales[..., :2])


@pytest.mark.parametrize("cache", ["4bit", "16bit"])
def test_a_captured_step_of_metadata_rotation_append_and_decode(cache):
    """One graph replayed step after step with the caller's own work between, against the same calls made eagerly."""

    require_gpu()
    from prism_infer.engine.step_metadata import build_step_metadata

    a, b = (RotaryRequests(4, 8, 2, BF16, cache, seed=3) for _ in range(2))
    for r in (a, b):
        new = [30, 1, 17, 64]
        m = r.metadata(new, sum(new))
        (q, k, v), _ = r.tokens(new, sum(new))
        r.prefill(q, k, v, m, cached_prefix=False)
    qkv = torch.zeros(4, 12 * 128, dtype=BF16, device="cuda")
    split = lambda: [t.unflatten(1, (-1, 128)) for t in qkv.split([8 * 128, 2 * 128, 2 * 128], 1)]  # noqa: E731
    state = [t.clone() for t in (a.tables, a.cached, a.start)]
    new = torch.ones(4, dtype=torch.int32, device="cuda")

    def step(layer, tables, cached, start):
        m = build_step_metadata(tables, cached, new, block_size=16, num_tokens=4, free_blocks=a.free, free_start=start)
        return m, layer(*split(), m)

    before = [None if c is None else c.clone() for c in a.caches]
    step(a.decode, *state)  # warm, on what is put back
    for c, old in zip(a.caches, before):
        if c is not None:
            c.view(torch.uint8).copy_(old.view(torch.uint8))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m, out = step(a.decode, *state)
    for lens in ([1, 1, 1, 1], [1, 0, 1, 1], [1, 1, 1, 0], [0, 0, 0, 0], [1, 1, 1, 1]):
        qkv.copy_(torch.randn(qkv.shape, generator=a.g))
        new.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got, rows = out.clone(), sum(lens)
        eager, want = step(b.decode, b.tables, b.cached, b.start)
        torch.cuda.synchronize()
        b.tables, b.cached, b.start = eager.block_tables, eager.context_lens, eager.next_free
        assert torch.equal(m.packed, eager.packed)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))
        assert all(same_bytes(x, y) for x, y in zip(a.caches, b.caches) if x is not None)
        assert rows == 0 or got[:rows].isfinite().all()
        for old, now in zip(state, (m.block_tables, m.context_lens, m.next_free)):
            old.copy_(now)


def test_two_graphs_and_an_eager_call_at_once():
    """Graphs captured one after the other share no scratch: replayed on two streams together they give what each gives alone."""

    require_gpu()
    from _fp4 import Pool
    from prism_infer.ops.paged_decode import paged_decode_attention

    pools = [Pool([9000, 300], page=16, kv_heads=2, dim=128, seed=31), Pool([100, 7000, 2500], page=64, kv_heads=2, dim=128, seed=32)]
    qs = [torch.randn(len(p.ctx), 8, 128, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i, p in enumerate(pools)]
    call = lambda i: paged_decode_attention(qs[i], pools[i].kc, pools[i].vc, pools[i].tables, pools[i].lens, 0.09,  # noqa: E731
                                            k_scale_cache=pools[i].ks, v_scale_cache=pools[i].vs)
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graphs[i].replay()
        eager = call(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[1])


def test_pages_behind_32_bit_offsets():
    """Blocks past 4 GiB of a 4-bit cache: rows appended, read back and attended as in a small one."""

    require_gpu()
    from prism_infer.ops.kv_cache_load import load_kvcache
    from prism_infer.ops.paged_decode import paged_decode_attention
    from prism_infer.ops.paged_prefill import paged_prefill_attention
    from prism_infer.ops.rotary_kv_store import rotate_store_kvcache
    from types import SimpleNamespace

    # 33000 blocks of 256 tokens of 8 heads of 64 bytes: 4.3e9 bytes of K and of V, and 33000 * 8192 exponents
    blocks, page, tokens = 33000, 256, 600
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(tokens, 24 * 128, generator=g).to(BF16).cuda()
    q, k, v = (t.unflatten(1, (8, 128)) for t in qkv.split(8 * 128, 1))
    big = [torch.empty(blocks, page, 8, n, dtype=torch.uint8, device="cuda") for n in (64, 64, 4, 4)]
    small = [t.view(torch.uint8) for p in (empty_cache((4, page, 8, 128)), empty_cache((4, page, 8, 128))) for t in p]
    small = [small[0], small[2], small[1], small[3]]
    cos_sin, positions = table(tokens, 128).cuda(), torch.arange(tokens, dtype=torch.int32, device="cuda")
    out = []
    for caches, ids in ((big, [blocks - 2, 32999, 32800]), (small, [1, 3, 0])):
        kc, vc, ks, vs = caches[0].view(FP4), caches[1].view(FP4), caches[2].view(E8M0), caches[3].view(E8M0)
        slots = (torch.tensor(ids)[torch.arange(tokens) // page] * page + torch.arange(tokens) % page).int().cuda()
        tables = torch.tensor([ids], dtype=torch.int32, device="cuda")
        turned = rotate_store_kvcache(q, k, v, cos_sin, positions, kc, vc, slots, ks, vs)
        key, value = load_kvcache(kc, vc, slots, ks, vs)
        context = SimpleNamespace(block_tables=tables, context_lens=torch.tensor([tokens], dtype=torch.int32, device="cuda"),
                                  cu_seqlens_q=torch.tensor([0, 200], dtype=torch.int32, device="cuda"))
        chunk = paged_prefill_attention(turned[-200:], kc, vc, context, num_heads=8, num_kv_heads=8, scale=0.09, k_scale_cache=ks,
                                        v_scale_cache=vs)
        one = paged_decode_attention(turned[-1:], kc, vc, tables, context.context_lens, 0.09, k_scale_cache=ks, v_scale_cache=vs)
        out.append((turned, key, value, chunk, one))
    for a, b in zip(*out):
        assert torch.equal(a, b) and not math.isnan(float(a.float().sum()))


def test_the_layer_refuses():
    require_gpu()
    r = RotaryRequests(2, 8, 2, BF16, "4bit")
    m = r.metadata([3, 3], 6)
    (q, k, v), _ = r.tokens([3, 3], 6)
    decode_meta = _as_decode(r.metadata([1, 1], 2))
    with pytest.raises(RuntimeError, match="requires the step's positions"):
        r.decode(q[:2], k[:2], v[:2], decode_meta)
    with pytest.raises(ValueError, match="positions must be"):
        r.prefill(q, k, v, m, m.positions[:5], cached_prefix=False)
    r.prefill.k_scale_cache = None
    with pytest.raises(RuntimeError, match="bound together"):
        r.prefill(q, k, v, m, cached_prefix=False)
    r.prefill.v_scale_cache = None
    with pytest.raises(ValueError, match="need their exponents"):
        r.prefill(q, k, v, m, cached_prefix=False)
    r.decode.cos_sin_cache = None
    with pytest.raises(RuntimeError, match="need a bound cos_sin_cache"):
        r.decode(q[:2], k[:2], v[:2], decode_meta, m.positions[:2])


def test_layers_without_a_rotation_over_4bit_caches():
    """The layers' plain store and attention over a 4-bit cache, as over the others."""

    require_gpu()
    r = RotaryRequests(3, 8, 2, BF16, "4bit")
    r.table = torch.cat([torch.ones(700, 64), torch.zeros(700, 64)], 1)  # the host's rotation turns nothing
    r.prefill.cos_sin_cache = r.decode.cos_sin_cache = None
    for new, prefix in (([20, 5, 33], False), ([7, 40, 1], True)):
        m = r.metadata(new, sum(new))
        (q, k, v), turned = r.tokens(new, sum(new))
        out = r.prefill(q, k.contiguous(), v.contiguous(), m, cached_prefix=prefix)
        r.compare(turned, out, new, own_keys=not prefix)
    m = r.metadata([1, 1, 1], 3)
    (q, k, v), turned = r.tokens([1, 1, 1], 3)
    r.compare(turned, r.decode(q, k.contiguous(), v.contiguous(), m), [1, 1, 1], own_keys=False, step=True)
