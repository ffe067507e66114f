"""What prompt attention, 16-bit paged prefill and step metadata refuse before any GPU work."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

BF16 = torch.bfloat16


def _prompt(q=(6, 4, 64), k=(6, 2, 64), v=None, cu=(0, 6), cu_k=None, heads=4, kv=2, dtype=BF16, kdtype=None, cdtype=torch.int32):
    from prism_infer.ops.prompt_attention import prompt_attention

    return prompt_attention(
        torch.zeros(q, dtype=dtype), torch.zeros(k, dtype=kdtype or dtype), torch.zeros(v or k, dtype=kdtype or dtype),
        torch.tensor(cu, dtype=cdtype), num_heads=heads, num_kv_heads=kv, scale=0.1,
        cu_seqlens_k=None if cu_k is None else torch.tensor(cu_k, dtype=torch.int32))


@pytest.mark.parametrize("kw,match", [
    (dict(heads=3), "divisible"), (dict(kv=0), "divisible"), (dict(q=(6, 256)), "q must be"), (dict(q=(6, 8, 64)), "q must be"),
    (dict(k=(6, 2, 32)), "k and v must be"), (dict(k=(6, 1, 64)), "k and v must be"), (dict(v=(5, 2, 64)), "k and v must be"),
    (dict(kdtype=torch.float16), "dtype mismatch"), (dict(cdtype=torch.int64), "torch.int32"), (dict(cu=()), "batch \\+ 1"),
    (dict(cu=((0, 6),)), "one-dimensional"), (dict(cu_k=(0, 3, 6)), "same length"), (dict(k=(7, 2, 64)), "same tokens"),
])
def test_prompt_attention_contract(kw, match):
    with pytest.raises(ValueError, match=match):
        _prompt(**kw)


def test_prompt_attention_takes_only_so_many_tokens():
    from prism_infer.ops.prompt_attention import MAX_PROMPT_TOKENS, prompt_attention

    x = torch.zeros(1, 1, 64, dtype=BF16).expand(MAX_PROMPT_TOKENS + 1, 1, 64)
    with pytest.raises(RuntimeError, match="at most"):
        prompt_attention(x, x, x, torch.tensor([0, 1], dtype=torch.int32), num_heads=1, num_kv_heads=1, scale=0.1)


def test_prompt_attention_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="runs on the GPU|not built|cannot load"):
        _prompt()


def test_paged_prefill_over_16_bit_caches_has_no_cpu_path_and_no_scales():
    from prism_infer.ops.paged_prefill import paged_prefill_attention

    cache = torch.zeros(2, 16, 2, 64, dtype=BF16)
    ctx = SimpleNamespace(block_tables=torch.zeros(1, 1, dtype=torch.int32), context_lens=torch.tensor([6], dtype=torch.int32),
                          cu_seqlens_q=torch.tensor([0, 6], dtype=torch.int32))
    q = torch.zeros(6, 4, 64, dtype=BF16)
    with pytest.raises(RuntimeError, match="runs on the GPU|not built|cannot load"):
        paged_prefill_attention(q, cache, cache, ctx, num_heads=4, num_kv_heads=2, scale=0.1)
    scales = torch.ones(2, 16, 2)
    with pytest.raises(ValueError, match="FP8"):
        paged_prefill_attention(q, cache, cache, ctx, num_heads=4, num_kv_heads=2, scale=0.1, k_scale_cache=scales,
                                v_scale_cache=scales)


def _meta(tables=(2, 3), cached=2, new=2, dtype=torch.int32, size=16, tokens=4, **kw):
    from prism_infer.engine.step_metadata import build_step_metadata

    return build_step_metadata(torch.zeros(tables, dtype=dtype), torch.zeros(cached, dtype=torch.int32),
                               torch.zeros(new, dtype=torch.int32), block_size=size, num_tokens=tokens, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(size=0), "positive"), (dict(tokens=-1), "not negative"), (dict(size=2**31), "below"),
    (dict(tokens=2**30 + 1), "at most"), (dict(tables=(2,)), "block_tables must be"),
    (dict(cached=3), "one entry per request"), (dict(new=1), "one entry per request"), (dict(dtype=torch.int64), "torch.int32"),
    (dict(free_blocks=torch.zeros(2, 2, dtype=torch.int32)), "one-dimensional"),
    (dict(free_start=torch.zeros(2, dtype=torch.int32)), "one value"),
])
def test_step_metadata_contract(kw, match):
    with pytest.raises(ValueError, match=match):
        _meta(**kw)


def test_step_metadata_has_no_cpu_path():
    with pytest.raises(RuntimeError, match="runs on the GPU|not built|cannot load"):
        _meta()


def test_abi_refuses_before_any_launch():
    """Bad geometry, layouts and null pointers come back as error codes with a message, not as a launch."""

    from prism_infer import _native

    if not _native.available():
        pytest.skip("the library is not built")
    lib = _native.lib()
    s3, s4 = _native.int64s(512, 128, 1), _native.int64s(4096, 512, 128, 1)
    p = 4096  # (never dereferenced)

    def prompt(**kw):
        a = dict(q=p, qs=s3, k=p, ks=s3, v=p, vs=s3, dtype=1, cq=p, ck=p, out=p, os=s3, batch=1, tq=4, tk=4, h=4, hk=4, d=128) | kw
        rc = lib.prism_prompt_attention(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["dtype"], a["cq"], a["ck"], a["out"],
                                        a["os"], a["batch"], a["tq"], a["tk"], a["h"], a["hk"], a["d"], 0.1, None, 0, None)
        return rc, lib.prism_last_error().decode()

    assert prompt(batch=-1)[0] == -1 and prompt(q=None)[0] == -1 and prompt(k=None)[0] == -1 and prompt(cq=None)[0] == -1
    assert prompt(h=6)[0] == -1
    assert prompt(dtype=0)[0] == -2 and prompt(dtype=3)[0] == -2 and prompt(d=96)[0] == -2
    assert prompt(q=p + 2)[0] == -2 and prompt(ks=_native.int64s(513, 128, 1))[0] == -2
    assert "span" in prompt(ks=_native.int64s(2**30, 128, 1))[1]
    assert "too many" in prompt(tq=2**31 - 1, h=8, hk=1)[1] and "too many" in prompt(tq=2**29 + 1)[1]
    assert "too many" in prompt(tq=2**28, h=64, hk=64)[1] and "too many" in prompt(tk=2**31 - 1)[1]
    assert prompt(tq=0, q=None, out=None)[0] == 0

    def paged(q_dtype=1, dtype=1, d=128, page=16, ks=None, h=4, status=p):
        rc = lib.prism_paged_prefill_ws(p, q_dtype, s3, p, p, dtype, s4, s4, ks, ks, s3, s3, p, _native.int64s(1, 1), p, p, p, s3,
                                        1, 4, h, 4, d, page, 2, 1, 0.1, status, None, 0, None, None)
        return rc, lib.prism_last_error().decode()

    assert paged(q_dtype=2)[0] == -2 and paged(ks=p)[0] == -2 and paged(d=32)[0] == -2 and paged(page=24)[0] == -2
    assert paged(h=6)[0] == -1 and paged(status=None)[0] == -1

    def meta(**kw):
        a = dict(bt=p, c=p, n=p, f=p, nf=1, b=1, w=1, size=16, t=4, out=p) | kw
        return lib.prism_step_metadata(a["bt"], _native.int64s(1, 1), a["c"], a["n"], a["f"], a["nf"], None, a["b"], a["w"],
                                       a["size"], a["t"], a["out"], None)

    assert meta(b=-1) == -1 and meta(size=0) == -1 and meta(c=None) == -1 and meta(bt=None) == -1 and meta(f=None) == -1
    assert meta(out=None) == -1 and meta(b=8193) == -2 and meta(out=p + 4) == -2
    assert lib.prism_step_metadata_words(3, 5, 7) == 2 * 8 + 12 + 15
