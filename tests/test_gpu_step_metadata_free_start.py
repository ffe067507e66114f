"""A free_start behind the free blocks: only a request that needs a block does not fit."""

from __future__ import annotations

import pytest
import torch

from _helpers import require_gpu

pytestmark = pytest.mark.gpu

FITS = 2**31 - 1


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("free,start", [([], 9), ([40, 41], 3), (None, 5), ([40, 41], 2)])
def test_requests_that_need_no_block_fit(free, start):
    require_gpu()
    from prism_infer.engine.step_metadata import build_step_metadata

    tables = _int32([[7, 8, -5], [3, -5, -5], [5, 6, -5], [9, -5, -5]])
    cached = _int32([20, 3, 31, 16])

    def step(new):
        return build_step_metadata(tables, cached, _int32(new), block_size=16, num_tokens=sum(new),
                                   free_blocks=None if free is None else _int32(free), free_start=_int32([start]))

    m = step([4, 1, 1, 0])
    assert m.check().next_free.item() == start and m.first_misfit.item() == FITS
    assert m.slot_mapping.tolist() == [8 * 16 + 4, 8 * 16 + 5, 8 * 16 + 6, 8 * 16 + 7, 3 * 16 + 3, 6 * 16 + 15]
    m = step([4, 1, 2, 1])  # the third needs a block, and so does the fourth
    assert m.first_misfit.item() == 2 and m.next_free.item() == start + 2
    assert m.slot_mapping.tolist()[-3:] == [6 * 16 + 15, -1, -1]
    with pytest.raises(RuntimeError, match="request 2 does not fit"):
        m.check()
