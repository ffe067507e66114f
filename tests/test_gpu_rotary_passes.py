"""Rotation with append where a wave has two and six passes of a token's rows: bit for bit, with last waves and passes that are
partly empty, and passes that hold queries, keys and values at once."""

from __future__ import annotations

import pytest
import torch

from _helpers import require_gpu
from test_gpu_rotary_store import test_rotation_and_append_match_the_definition as rotation_and_append

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# passes of a wave; tokens, q heads, kv heads, dim, rotary, pairs, axes, input, cache, row padding
CASES = [
    (2, (1000, 32, 8, 128, 128, False, 1, BF16, "fp4", 0)),
    (2, (1001, 32, 8, 128, 64, True, 3, BF16, "fp8", 64)),
    (2, (900, 28, 4, 128, 128, False, 1, F16, "f16", 0)),    # nine passes
    (2, (2050, 12, 3, 64, 64, False, 1, BF16, "fp4", 8)),    # three
    (2, (1400, 8, 2, 256, 128, False, 3, F32, "fp4", 0)),
    (6, (4100, 3, 1, 128, 128, True, 1, F16, "fp8_unit", 0)),  # two, the second of one row
    (6, (2100, 32, 8, 128, 128, False, 3, BF16, "fp4", 0)),
    (6, (2101, 28, 4, 128, 96, False, 1, BF16, "fp8", 8)),   # nine
    (6, (2049, 28, 4, 128, 128, True, 1, F16, "fp4", 0)),
    (6, (4100, 12, 3, 64, 32, True, 1, F16, "bf16", 0)),     # three
    (6, (4097, 8, 2, 256, 256, False, 1, F32, "f32", 0)),
    (6, (4096, 20, 5, 64, 64, False, 1, BF16, "bf16", 16)),  # four
]


def passes_of_a_wave(tokens, q_heads, heads, dim, enough=16 * 256):
    passes = -(-(q_heads + 2 * heads) // (512 // dim))
    return next(n for n in (6, 2, 1) if n == 1 or tokens * -(-passes // n) >= enough)


@pytest.mark.parametrize("passes,case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c) if isinstance(c, tuple) else str(c))
def test_passes(passes, case):
    require_gpu()
    assert passes_of_a_wave(*case[:4]) == passes
    rotation_and_append(case)
