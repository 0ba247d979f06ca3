"""Attention of the paged 4-bit cache at the ends of its number ranges: rows of
zeros and tiny rows under tiny scales, rows as large and as small as their type
holds, and scores whose products are far larger than their sums.

Bounds are those of test_gpu_kv4.check_attn unless a test derives its own."""
import numpy as np
import pytest

import kv4_ref as R
import zero_b200 as zb
from test_gpu_kv4 import HD, NONE, TYPES, cache, check_attn, make, run_attn, store

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq", [1, 3, 140])
@pytest.mark.parametrize("scale", [1e-10, 9e-16, 1e-30, 1e-38])
def test_zero_and_tiny_rows_under_a_tiny_scale(ctx, dtype, nq, scale):
    """Scores of nearly 0: a row's result is the mean of the values that it sees."""
    c = make(ctx, 40 + nq, [300, nq + 2], [nq, nq], 4, 2, 16)
    c["q"][0] = 0
    c["q"][nq:, 1] = 0
    c["q"][nq // 2, 2] *= 1e-5 if dtype == "f16" else 2.0 ** -100
    o, q = run_attn(c, dtype, scale)
    check_attn(c, o, q, dtype, float(np.float32(scale)))
    c["kv"].check()
    c["kv"].close()
