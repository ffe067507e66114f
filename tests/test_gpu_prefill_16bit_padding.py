"""A captured chunk over 16-bit pages whose rows are padded: the rows outside the sequences are 0 on every replay."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _attention16 import assert_within, attention64
from _helpers import require_gpu

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,dim,page,heads,prefix", [(BF16, 128, 64, 8, 900), (F16, 64, 16, 6, 30), (BF16, 64, 256, 2, 5000)])
def test_padding_of_the_op(dtype, dim, page, heads, prefix):
    require_gpu()
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    rows, kv_heads, keys = 300, 2, prefix + 128
    pages = -(-keys // page)
    g = torch.Generator().manual_seed(dim + page)
    q = torch.randn(rows, heads, dim, generator=g).to(dtype)
    k, v = (torch.randn(2, pages * page, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    caches = [x.view(2 * pages, page, kv_heads, dim).cuda() for x in (k, v)]
    context = SimpleNamespace(block_tables=torch.arange(2 * pages, dtype=torch.int32, device="cuda").view(2, pages),
                              context_lens=_int32([keys, keys]), cu_seqlens_q=_int32([0, 1, 2]))
    dq = q.cuda()

    def call():
        return paged_prefill_attention(dq, *caches, context, num_heads=heads, num_kv_heads=kv_heads, scale=0.1)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for cu in ([0, 1, 2], [5, 105, 233], [0, 128, 256], [172, 173, 300], [0, 100, 128]):
        context.cu_seqlens_q.copy_(_int32(cu))
        out.fill_(float("nan"))
        graph.replay()
        assert (out[:cu[0]] == 0).all() and (out[cu[2]:] == 0).all(), cu
        for i in range(2):
            want, bound = attention64(q[cu[i]:cu[i + 1]], k[i, :keys], v[i, :keys], 0.1)
            assert_within(out[cu[i]:cu[i + 1]], want, bound, f"{cu} {i}")
        assert torch.equal(call(), out[cu[0]:cu[2]])


def test_padding_of_a_layers_step():
    """Metadata, store and attention behind a cached prefix in one graph, its rows padded."""

    require_gpu()
    from prism_infer.engine.prefill_attention import PagedKVPrefillAttention
    from prism_infer.engine.step_metadata import build_step_metadata

    rows, page, batch = 128, 16, 3
    g = torch.Generator().manual_seed(9)
    layer = PagedKVPrefillAttention(8, 2, 128, 0.1)
    old_k, old_v = (torch.randn(batch * 10, page, 2, 128, generator=g).to(BF16) for _ in range(2))
    layer.k_cache, layer.v_cache = old_k.cuda(), old_v.cuda()
    tables = torch.full((batch, 20), -1, dtype=torch.int32)
    tables[:, :5] = torch.arange(batch * 5, dtype=torch.int32).view(batch, 5)
    cached, free, new = _int32([70, 80, 65]), torch.arange(15, 30, dtype=torch.int32, device="cuda"), _int32([1, 1, 1])
    q, k, v = (torch.randn(rows, h, 128, generator=g).to(BF16) for h in (8, 2, 2))
    dq, dk, dv, dt = q.cuda(), k.cuda(), v.cuda(), tables.cuda()

    def step():
        m = build_step_metadata(dt, cached, new, block_size=page, num_tokens=rows, free_blocks=free)
        return layer(dq, dk, dv, m, cached_prefix=True)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lens in ([1, 1, 1], [40, 3, 60], [30, 50, 48]):
        new.copy_(_int32(lens))
        out.fill_(float("nan"))
        graph.replay()
        at = 0
        for i, n in enumerate(lens):
            have = cached[i].item()
            keys, values = (torch.cat([old[tables[i, :5].long()].flatten(0, 1)[:have], x[at:at + n]])
                            for old, x in ((old_k, k), (old_v, v)))
            assert_within(out[at:at + n], *attention64(q[at:at + n], keys, values, 0.1), f"{lens} {i}")
            at += n
        assert (out[at:] == 0).all(), lens
