"""Tables that are columns of a wider buffer: rows start on 16 bytes, their lengths are no multiple of four entries."""

from __future__ import annotations

import pytest
import torch

from _helpers import require_gpu
from test_gpu_step_metadata import _same, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pitch,first,width", [(8, 0, 7), (8, 0, 6), (8, 0, 5), (12, 4, 7), (16, 0, 9), (8, 0, 8), (8, 1, 7), (12, 2, 8)])
def test_columns_of_a_wider_buffer(pitch, first, width):
    require_gpu()
    from prism_infer.engine.step_metadata import build_step_metadata

    page, batch = 16, 50
    g = torch.Generator().manual_seed(pitch + width)
    buffer = torch.randint(-9, 10**6, (batch, pitch), generator=g, dtype=torch.int32)
    cached = torch.randint(0, page * width - 20, (batch,), generator=g).tolist()
    new = torch.randint(0, 20, (batch,), generator=g).tolist()
    for i, c in enumerate(cached):
        buffer[i, first:first + -(-c // page)] = torch.randint(0, 10**6, (-(-c // page),), generator=g, dtype=torch.int32)
    tables, free = buffer[:, first:first + width], list(range(2 * batch))
    case = (tables, cached, new, page, sum(new) + 3, free)
    cuda = buffer.cuda()[:, first:first + width]
    assert cuda.stride() == (pitch, 1)
    x = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in (cached, new, free)]
    m = build_step_metadata(cuda, x[0], x[1], block_size=page, num_tokens=case[4], free_blocks=x[2])
    _same(m.check(), plain(*case))
