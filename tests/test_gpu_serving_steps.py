"""Prompts, a chunk behind them and decode steps of one layer, all from the requests' lengths on the device.

Every step's output is compared with plain attention in 64 bits over the tokens so far.  16-bit caches keep the bounds
of _attention16; a step's decode op has the reference's bound (2e-2, tests/_helpers.py).  Over a scaled FP8 cache what
was stored is read back and dequantised, so that only attention is compared.
"""

from __future__ import annotations

import pytest
import torch

from _attention16 import assert_within, attention64
from _helpers import require_gpu

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


class Requests:
    """What a server knows: each request's tokens so far (K, V), and the device's metadata."""

    def __init__(self, batch, heads, kv_heads, dtype, cache, page=16, pool=160, seed=1):
        from prism_infer.engine.decode_attention import PagedKVDecodeAttention
        from prism_infer.engine.prefill_attention import PagedKVPrefillAttention

        self.g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dtype, self.page, self.batch = heads, kv_heads, dtype, page, batch
        self.scale = 128 ** -0.5
        self.prefill = PagedKVPrefillAttention(heads, kv_heads, 128, self.scale)
        self.decode = PagedKVDecodeAttention(heads, kv_heads, 128, self.scale)
        kind = torch.float8_e4m3fn if cache == "scaled" else dtype
        caches = [torch.zeros(pool, page, kv_heads, 128, dtype=kind, device="cuda") for _ in range(2)]
        scales = [torch.ones(pool, page, kv_heads, device="cuda") for _ in range(2)] if cache == "scaled" else [None, None]
        for layer in (self.prefill, self.decode):
            layer.k_cache, layer.v_cache = caches
            layer.k_scale_cache, layer.v_scale_cache = scales
        self.free = torch.randperm(pool, generator=self.g).to(torch.int32).cuda()
        self.tables = torch.full((batch, 40), -1, dtype=torch.int32, device="cuda")
        self.cached = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.start = None
        self.k, self.v = ([torch.zeros(0, kv_heads, 128, dtype=dtype)] * batch for _ in range(2))

    def metadata(self, new, rows):
        from prism_infer.engine.step_metadata import build_step_metadata

        m = build_step_metadata(self.tables, self.cached, torch.tensor(new, dtype=torch.int32, device="cuda"), block_size=self.page,
                                num_tokens=rows, free_blocks=self.free, free_start=self.start).check()
        self.tables, self.cached, self.start = m.block_tables, m.context_lens, m.next_free
        return m

    def tokens(self, new, rows):
        q, k, v = (torch.randn(rows, h, 128, generator=self.g).to(self.dtype) for h in (self.heads, self.kv_heads, self.kv_heads))
        at = 0
        for i, n in enumerate(new):
            self.k[i], self.v[i] = torch.cat([self.k[i], k[at:at + n]]), torch.cat([self.v[i], v[at:at + n]])
            at += n
        return q, k, v

    def stored(self, i):
        """Request i's tokens as its pages hold them, dequantised."""

        pages = self.tables[i, :-(-self.k[i].shape[0] // self.page)].long()
        pairs = ((self.decode.k_cache, self.decode.k_scale_cache), (self.decode.v_cache, self.decode.v_scale_cache))
        rows = [c.view(torch.uint8)[pages].view(c.dtype).flatten(0, 1)[:self.k[i].shape[0]].cpu().double() for c, _ in pairs]
        if pairs[0][1] is not None:
            rows = [r * s[pages].flatten(0, 1)[:r.shape[0], :, None].cpu().double() for r, (_, s) in zip(rows, pairs)]
        return rows


def _compare(r, q, got, new, *, exact_keys, loose=None):
    at = 0
    for i, n in enumerate(new):
        if n:
            k, v = (r.k[i], r.v[i]) if exact_keys else r.stored(i)
            want, bound = attention64(q[at:at + n], k, v, r.scale)
            assert_within(got[at:at + n], want, bound if loose is None else torch.full_like(bound, loose), f"request {i}")
        at += n


@pytest.mark.parametrize("cache,dtype", [("16bit", BF16), ("16bit", F16), ("scaled", BF16)])
def test_prompts_chunk_and_decode_steps(cache, dtype):
    require_gpu()
    r = Requests(5, 8, 2, dtype, cache)
    plain = cache == "16bit"
    # prompts, padded to 256 rows
    new = [37, 1, 64, 90, 17]
    m = r.metadata(new, 256)
    q, k, v = r.tokens(new, 256)
    out = r.prefill(q.cuda(), k.cuda(), v.cuda(), m, cached_prefix=False)
    _compare(r, q, out, new, exact_keys=True)
    assert (out[sum(new):] == 0).all()
    if plain:  # what the pages hold is what was passed
        for i in range(r.batch):
            assert torch.equal(r.stored(i)[0], r.k[i].double()) and torch.equal(r.stored(i)[1], r.v[i].double())
    # a chunk behind each of them
    new = [100, 3, 64, 1, 45]
    m = r.metadata(new, sum(new))
    q, k, v = r.tokens(new, sum(new))
    out = r.prefill(q.cuda(), k.cuda(), v.cuda(), m, cached_prefix=True)
    _compare(r, q, out, new, exact_keys=False, loose=None if plain else 2e-2)
    # decode steps
    for _ in range(20):
        new = [1] * r.batch
        m = r.metadata(new, r.batch)
        q, k, v = r.tokens(new, r.batch)
        out = r.decode(q.cuda(), k.cuda(), v.cuda(), m)
        _compare(r, q, out, new, exact_keys=False, loose=2e-2)


def test_prefill_step_captured_with_lengths_of_the_replay():
    """Metadata, store and prompt attention of a padded batch in one graph, replayed with other lengths and tokens."""

    require_gpu()
    from prism_infer.engine.step_metadata import build_step_metadata

    r = Requests(4, 8, 2, BF16, "16bit")
    rows = 192
    q, k, v = (torch.zeros(rows, h, 128, dtype=BF16, device="cuda") for h in (8, 2, 2))
    new = torch.zeros(4, dtype=torch.int32, device="cuda")

    def step():
        m = build_step_metadata(r.tables, r.cached, new, block_size=16, num_tokens=rows, free_blocks=r.free)
        return m, r.prefill(q, k, v, m, cached_prefix=False)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m, out = step()
    for lens in ([10, 80, 0, 33], [64, 64, 64, 0], [1, 1, 1, 1], [0, 0, 0, 0]):
        r.k, r.v = ([torch.zeros(0, 2, 128, dtype=BF16)] * 4 for _ in range(2))
        hq, hk, hv = r.tokens(lens, rows)
        for device, host in ((q, hq), (k, hk), (v, hv)):
            device.copy_(host)
        new.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        _compare(r, hq, out, lens, exact_keys=True)
        assert (out[sum(lens):] == 0).all() and m.slot_mapping[sum(lens):].eq(-1).all()
        slots = m.slot_mapping[:sum(lens)].long()
        assert torch.equal(r.prefill.k_cache.flatten(0, 1)[slots].cpu(), hk[:sum(lens)])


def test_metadata_that_the_layer_refuses():
    require_gpu()
    r = Requests(2, 8, 2, BF16, "16bit")
    m = r.metadata([3, 3], 6)
    q, k, v = (x.cuda() for x in r.tokens([3, 3], 6))
    r.prefill.k_cache = torch.tensor([])
    with pytest.raises(RuntimeError, match="bound together"):
        r.prefill(q, k, v, m, cached_prefix=False)
