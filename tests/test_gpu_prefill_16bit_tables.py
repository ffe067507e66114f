"""16-bit paged prefill over tables without columns and caches without pages: the reference's errors."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _helpers import require_gpu

pytestmark = pytest.mark.gpu


def _inputs(tables, *, pages=4, dim=64, page=16):
    """Two requests of six and three tokens, nothing in front of them."""

    q = torch.ones(9, 4, dim, dtype=torch.bfloat16, device="cuda")
    cache = torch.ones(pages, page, 2, dim, dtype=torch.bfloat16, device="cuda")
    return q, cache, SimpleNamespace(block_tables=tables, context_lens=torch.tensor([6, 3], dtype=torch.int32, device="cuda"),
                                     cu_seqlens_q=torch.tensor([0, 6, 9], dtype=torch.int32, device="cuda"))


def _call(q, cache, context):
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    return paged_prefill_attention(q, cache, cache, context, num_heads=4, num_kv_heads=2, scale=0.1)


def _raises(match, *inputs):
    for _ in range(3):  # (a stream's first call is checked in Python, later ones by the native path)
        with pytest.raises(RuntimeError, match=match):
            _call(*inputs)


@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128)])
def test_tables_without_columns(page, dim):
    require_gpu()
    whole = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    assert (_call(*_inputs(whole, page=page, dim=dim)) == 1).all()
    for tables in (torch.zeros(2, 0, dtype=torch.int32, device="cuda"), whole[:, :0]):
        _raises("invalid block table for paged KV reference: context_len=6, remaining=6", *_inputs(tables, page=page, dim=dim))
    assert (_call(*_inputs(whole, page=page, dim=dim)) == 1).all()


def test_a_step_whose_tables_have_no_columns():
    require_gpu()
    from prism_infer.engine.step_metadata import build_step_metadata

    q, cache, context = _inputs(torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
    new = context.context_lens
    m = build_step_metadata(context.block_tables, torch.zeros_like(new), new, block_size=16, num_tokens=9)
    _raises("invalid block table", q, cache, m)


def test_caches_without_pages():
    require_gpu()
    _raises("exceeds cache capacity", *_inputs(torch.zeros(2, 1, dtype=torch.int32, device="cuda"), pages=0))


def test_captured_without_columns():
    """Under capture nothing is reported; a call after it is as ever."""

    require_gpu()
    empty = _inputs(torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(*empty)
    for _ in range(2):
        graph.replay()
        assert out.shape == (9, 4, 64)
        assert (_call(*_inputs(torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda"))) == 1).all()
