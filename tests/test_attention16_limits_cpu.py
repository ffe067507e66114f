"""The largest calls of attention over 16-bit keys: what is documented is what is refused, before any launch."""

from __future__ import annotations

import pytest

WORKGROUPS = 2**24  # of 256 threads: a launch holds fewer


@pytest.fixture
def native():
    from prism_infer import _native

    if not _native.available():
        pytest.skip("the library is not built")
    return _native.lib(), _native.int64s


def _prompt(native, tokens, heads, kv_heads, batch):
    lib, int64s = native
    p, s = 4096, int64s(512, 128, 1)  # (never dereferenced)
    rc = lib.prism_prompt_attention(p, s, p, s, p, s, 1, p, p, p, s, batch, tokens, tokens, heads, kv_heads, 128, 0.1, None, 0, None)
    return rc, lib.prism_last_error().decode()


def _paged(native, tokens, heads, kv_heads, batch):
    lib, int64s = native
    p, s3, s4 = 4096, int64s(512, 128, 1), int64s(4096, 512, 128, 1)
    rc = lib.prism_paged_prefill_ws(p, 1, s3, p, p, 1, s4, s4, None, None, s3, s3, p, int64s(1, 1), p, p, p, s3, batch, tokens,
                                    heads, kv_heads, 128, 16, 2, 1, 0.1, p, None, 0, None, None)
    return rc, lib.prism_last_error().decode()


@pytest.mark.parametrize("call", [_prompt, _paged])
@pytest.mark.parametrize("tokens,heads,kv_heads,batch", [
    (2**29 // 8 + 1, 8, 1, 1),                         # rows of a kv head
    (128 * (WORKGROUPS // 64 - 2), 64, 64, 1),         # workgroups: blocks of 128 rows
    (128, 64, 64, WORKGROUPS // 64 - 2),               # and one per sequence
])
def test_too_many_rows_or_workgroups(native, call, tokens, heads, kv_heads, batch):
    rc, message = call(native, tokens, heads, kv_heads, batch)
    assert rc == -1 and "too many query rows" in message, (rc, message)
