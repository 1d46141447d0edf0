"""The paged cache where its data is unusual: scales of zero and of no use, table entries that name no
page, padded rows, overlapping memory, other streams, autograd.

Attention is held to the bounds of test_gpu_kvcache.py: the output's rounding, 2^-11 + 2^-13 of
sum p|v| and 1e-6; lse to 2e-5 of max(1, |lse|).
"""
from __future__ import annotations

import math

import pytest

from test_gpu_kvcache import check_attend, ints, make_cache, rope_table, row_starts

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------- scales
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("zero", [0.0, -0.0, 1e-44, 1e-30])
def test_value_scales_of_zero_keep_their_weight(cuda, dtype, D, zero):
    """A block whose value scale is zero (or too small for f32's reciprocals) holds values of zero: its keys
    keep their share of the softmax. On tiles with and without masked keys, whatever its codes."""
    def some(cache, rows, q):
        for row in rows:
            for page in row[:8:2]:
                cache.v_scale[0, page] = zero
            cache.v_scale[0, row[4], 0] = 0.5  # one head of a page only
    check_attend(cuda, [1, 1, 1], [333, 40, 256], 2, 4, D, 32, dtype, seed=D, tamper=some, with_starts=False)
    check_attend(cuda, [5, 300, 130], [400, 512, 300], 2, 4, D, 32, dtype, seed=D, tamper=some)
    check_attend(cuda, [200], [700], 1, 4, D, 64, dtype, seed=D, tamper=some, causal=False)


def test_value_scales_of_zero_everywhere(cuda):
    def none(cache, rows, q):
        cache.v_scale.zero_()
    def both(cache, rows, q):
        cache.v_scale.zero_()
        cache.k_scale.zero_()
    for tamper in (none, both):
        check_attend(cuda, [1, 1], [300, 17], 2, 4, 128, 32, seed=1, tamper=tamper, with_starts=False)
        check_attend(cuda, [300, 20], [300, 600], 2, 4, 128, 32, "bf16", seed=1, tamper=tamper)


def test_value_scales_far_apart(cuda):
    """Zero blocks beside small, ordinary and large ones in one row."""
    def uneven(cache, rows, q):
        for row in rows:
            for i, s in enumerate((0.0, 1e-18, 1e-12, 1e-3, 30.0, 0.0)):
                cache.v_scale[0, row[i]] = s
    check_attend(cuda, [1, 60], [300, 300], 2, 4, 128, 32, seed=8, tamper=uneven)
    check_attend(cuda, [280], [400], 2, 4, 128, 32, "bf16", seed=8, tamper=uneven)
