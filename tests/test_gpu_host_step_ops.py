"""Prompt attention, 16-bit paged prefill and step metadata through the native checks and through Python: the same results.

The native functions take a call or return None; what they return None for is handled, or refused with its message, in
Python.
"""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from _helpers import require_gpu

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _modules():
    import prism_infer.engine.step_metadata as meta
    import prism_infer.ops.paged_prefill as paged
    import prism_infer.ops.prompt_attention as prompt

    return prompt, paged, meta


@pytest.fixture
def host(monkeypatch):
    """Counts the native functions' answers; python() takes the Python path."""

    require_gpu()
    prompt, paged, meta = _modules()
    if prompt._HOST is None:
        pytest.skip("the native host path is not built")
    taken = {"prompt": 0, "prefill": 0, "step_metadata": 0}

    def counted(name):
        def call(*args):
            done = getattr(real, name)(*args)
            taken[name] += done is not None
            return done
        return call

    real = prompt._HOST
    fake = SimpleNamespace(**{name: counted(name) for name in taken})
    for m in (prompt, paged, meta):
        monkeypatch.setattr(m, "_HOST", fake)

    def python(run):
        with monkeypatch.context() as m:
            for module in (prompt, paged, meta):
                m.setattr(module, "_HOST", None)
            return run()

    return SimpleNamespace(taken=taken, python=python)


def _qkv(dtype=BF16, dim=128, tokens=70):
    g = torch.Generator(device="cuda").manual_seed(5)
    return [torch.randn(tokens, h, dim, generator=g, device="cuda", dtype=dtype) for h in (8, 2, 2)]


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (torch.float16, 64)])
def test_prompt(host, dtype, dim):
    prompt, _, _ = _modules()
    q, k, v = _qkv(dtype, dim)
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    other = torch.tensor([0, 20, 65], dtype=torch.int32, device="cuda")

    def call(q=q, k=k, v=v, cu=cu, **kw):
        return prompt.prompt_attention(q, k, v, cu, num_heads=8, num_kv_heads=2, scale=0.1, **kw)

    call()  # (the first on a device loads the kernels)
    host.taken["prompt"] = 0
    for run in (call, lambda: call(cu_seqlens_k=other), lambda: call(q=q[:, :, :].as_strided((1, 8, dim), (3, dim, 1)), k=k[:1],
                                                                      v=v[:1], cu=cu.new_tensor([0, 1]))):
        assert torch.equal(run(), host.python(run))
    assert host.taken["prompt"] == 3
    # not taken, the same results: rows off their 16 bytes, a scale that is no float, offsets with a stride
    odd = torch.empty(70, 8, dim + 1, dtype=dtype, device="cuda")[..., 1:].copy_(q)
    wide = torch.stack([cu, cu], dim=1)[:, 0]
    want = call()
    host.taken["prompt"] = 0
    assert torch.equal(call(q=odd), want) and torch.equal(call(cu=wide), want)
    assert torch.equal(prompt.prompt_attention(q, k, v, cu, num_heads=8, num_kv_heads=2, scale=1),
                       host.python(lambda: prompt.prompt_attention(q, k, v, cu, num_heads=8, num_kv_heads=2, scale=1.0)))
    assert host.taken["prompt"] == 0
    for bad in (dict(k=k[:60]), dict(v=v[:, :1]), dict(cu=cu.long()), dict(q=q[:, :6]), dict(k=k.to(torch.float32))):
        with pytest.raises((ValueError, RuntimeError)) as native:
            call(**bad)
        with pytest.raises(type(native.value)) as python:
            host.python(lambda: call(**bad))
        assert str(native.value) == str(python.value)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (torch.float16, 64)])
def test_paged(host, dtype, dim):
    _, paged, _ = _modules()
    q, _, _ = _qkv(dtype, dim)
    g = torch.Generator(device="cuda").manual_seed(6)
    k, v = (torch.randn(12, 32, 2, dim, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    tables = torch.tensor([[3, 1, 9, 4], [0, 2, 5, 11]], dtype=torch.int32, device="cuda")
    ctx = SimpleNamespace(block_tables=tables, context_lens=torch.tensor([110, 60], dtype=torch.int32, device="cuda"),
                          cu_seqlens_q=torch.tensor([0, 40, 70], dtype=torch.int32, device="cuda"))

    def call(q=q, k=k, v=v):
        return paged.paged_prefill_attention(q, k, v, ctx, num_heads=8, num_kv_heads=2, scale=0.1)

    call()
    host.taken["prefill"] = 0
    assert torch.equal(call(), host.python(call)) and host.taken["prefill"] == 1
    odd = torch.empty(70, 8, dim + 1, dtype=dtype, device="cuda")[..., 1:].copy_(q)
    assert torch.equal(call(q=odd), call())
    for bad in (dict(q=q.to(torch.float32)), dict(v=v.to(torch.float32)), dict(k=k[:5])):
        with pytest.raises((ValueError, RuntimeError)) as native:
            call(**bad)
        with pytest.raises(type(native.value)) as python:
            host.python(lambda: call(**bad))
        assert str(native.value) == str(python.value)
    tables[1, 1] = 99
    with pytest.raises(RuntimeError, match="exceeds cache capacity"):
        call()
    tables[1, 1] = 2
    assert torch.equal(call(), host.python(call))


@pytest.mark.parametrize("batch,page,longest", [(1, 16, 9000), (3, 64, 700), (300, 16, 60), (600, 32, 40)])
def test_paged_outcome_is_known_before_the_result(host, batch, page, longest):
    """The metadata's check sees every length and every needed block id, and no other; good calls follow one another."""

    _, paged, _ = _modules()
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(1, longest + 1, (batch,), generator=g)
    lens[batch // 2] = longest
    width = -(-longest // page) + 2
    k, v = (torch.randn(64, page, 1, 64, generator=g).to(BF16).cuda() for _ in range(2))
    q = torch.randn(batch, 2, 64, generator=g).to(BF16).cuda()
    tables = torch.randint(0, 64, (batch, width), generator=g, dtype=torch.int32)
    tables.masked_fill_(torch.arange(width)[None, :] >= -(-lens[:, None] // page), 10**6)  # (not needed: anything)
    good, good_lens = tables.cuda(), lens.int().cuda()
    ctx = SimpleNamespace(block_tables=good.clone(), context_lens=good_lens.clone(),
                          cu_seqlens_q=torch.arange(batch + 1, dtype=torch.int32, device="cuda"))

    def call():
        return paged.paged_prefill_attention(q, k, v, ctx, num_heads=2, num_kv_heads=1, scale=0.1)

    want = host.python(call)
    call()
    host.taken["prefill"] = 0
    outs = [call() for _ in range(20)]
    assert all(torch.equal(o, want) for o in outs) and host.taken["prefill"] == 20
    for seq in {0, batch // 2, batch - 1}:
        last = -(-int(lens[seq]) // page) - 1
        for entry in {0, last}:
            for bad in (-1, 64):
                ctx.block_tables[seq, entry] = bad
                with pytest.raises(RuntimeError, match="exceeds cache capacity|invalid block table"):
                    call()
                ctx.block_tables.copy_(good)
        for bad in (0, width * page + 1):
            ctx.context_lens[seq] = bad
            with pytest.raises(RuntimeError, match="invalid paged prefill lengths|invalid block table|exceeds cache capacity"):
                call()
            ctx.context_lens.copy_(good_lens)
        assert torch.equal(call(), want)
    assert torch.equal(call(), want)


def test_metadata(host):
    _, _, meta = _modules()
    tables = torch.arange(40, dtype=torch.int32, device="cuda").view(5, 8)
    cached = torch.tensor([0, 17, 33, 5, 0], dtype=torch.int32, device="cuda")
    new = torch.tensor([9, 1, 40, 0, 3], dtype=torch.int32, device="cuda")
    free = torch.arange(100, 140, dtype=torch.int32, device="cuda")

    def call(tables=tables, cached=cached, tokens=60, **kw):
        return meta.build_step_metadata(tables, cached, new, block_size=16, num_tokens=tokens, **({"free_blocks": free} | kw))

    def same(run):
        a, b = run(), host.python(run)
        for name in ("slot_mapping", "positions", "cu_seqlens_q", "context_lens", "max_context_len", "next_free", "first_misfit",
                     "block_tables"):
            x, y = getattr(a, name), getattr(b, name)
            assert torch.equal(x, y) and x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride(), name
            assert x.is_contiguous() and x.untyped_storage().data_ptr() == a.packed.untyped_storage().data_ptr()

    call()
    host.taken["step_metadata"] = 0
    same(call)
    same(lambda: call(free_start=free.new_tensor([3])))
    same(lambda: call(tables=tables.t().contiguous().t()))
    same(lambda: call(free_blocks=None))
    same(lambda: call(tokens=3))
    assert host.taken["step_metadata"] == 5
    out = call()
    same(lambda: call(out=out))
    for bad in (dict(cached=cached[:4]), dict(tables=tables.long()), dict(tokens=-1)):
        with pytest.raises(ValueError) as native:
            call(**bad)
        with pytest.raises(ValueError) as python:
            host.python(lambda: call(**bad))
        assert str(native.value) == str(python.value)
