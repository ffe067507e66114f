"""Calls over 4-bit caches that are too large for one launch: refused under their own name, before anything is read."""

from __future__ import annotations

import pytest
from test_fp4_cpu import P, attention, native  # noqa: F401  (the fixture)


@pytest.mark.parametrize("change", [dict(total=2 ** 30, batch=1), dict(total=2 ** 28 + 1, heads=4, kv_heads=2), dict(total=2 ** 24, heads=64, kv_heads=1)])
def test_chunks_of_too_many_rows(native, change):  # noqa: F811
    rc, message = attention(*native, cu=P, status=P, max_ctx=None, **change)
    assert rc < 0 and message == "prism_paged_fp4: too many query rows for one launch", (rc, message)
