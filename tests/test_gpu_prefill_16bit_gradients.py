"""Paged prefill over 16-bit caches refuses inputs whose gradients are recorded, as prompt attention does."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _helpers import require_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_gradients_are_refused_where_recorded(name):
    require_gpu()
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    x = dict(q=torch.ones(5, 4, 64, dtype=torch.bfloat16, device="cuda"),
             k=torch.ones(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda"), v=torch.ones(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda"))
    context = SimpleNamespace(block_tables=torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"),
                              context_lens=torch.tensor([20], dtype=torch.int32, device="cuda"),
                              cu_seqlens_q=torch.tensor([0, 5], dtype=torch.int32, device="cuda"))

    def call():
        return paged_prefill_attention(x["q"], x["k"], x["v"], context, num_heads=4, num_kv_heads=2, scale=0.1)

    assert (call() == 1).all()
    x[name].requires_grad_()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    with torch.no_grad():
        assert (call() == 1).all() and not call().requires_grad
