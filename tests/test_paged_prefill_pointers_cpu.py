"""Null pointers that a 16-bit paged prefill would read come back as error codes, not as a launch."""

from __future__ import annotations

import pytest

ARRAYS = ("q", "k", "v", "bt", "ctx", "cu", "out")


def _call(lib, int64s, **kw):
    p = 4096  # (never dereferenced)
    a = dict(q=p, k=p, v=p, bt=p, ctx=p, cu=p, out=p, batch=1, tokens=4, pages=2, width=1) | kw
    s3, s4 = int64s(512, 128, 1), int64s(4096, 512, 128, 1)
    rc = lib.prism_paged_prefill_ws(a["q"], 1, s3, a["k"], a["v"], 1, s4, s4, None, None, s3, s3, a["bt"], int64s(1, 1), a["ctx"],
                                    a["cu"], a["out"], s3, a["batch"], a["tokens"], 4, 4, 128, 16, a["pages"], a["width"], 0.1, p,
                                    None, 0, None, None)
    return rc, lib.prism_last_error().decode()


@pytest.fixture
def native():
    from prism_infer import _native

    if not _native.available():
        pytest.skip("the library is not built")
    return _native.lib(), _native.int64s


@pytest.mark.parametrize("name", ARRAYS)
def test_a_null_array_is_refused(native, name):
    rc, message = _call(*native, **{name: None})
    assert rc == -1 and "null argument" in message, (rc, message)


@pytest.mark.parametrize("empty", [dict(batch=0), dict(tokens=0)])
def test_without_rows_nothing_is_read(native, empty):
    assert _call(*native, **empty, **dict.fromkeys(ARRAYS))[0] == 0
