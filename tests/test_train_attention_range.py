"""Attention with its gradient on values far from 1 (n3d_attention_forward, n3d_attention_backward), against 64
bits within the bounds derived in test_train_attention.py."""

import pytest

from test_train_attention import TYPES, run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("std", [1e-20, 1e-30])
def test_tiny_queries_and_keys_attend_evenly(dtype, hd, std):
    run(1, 130, 200, 2, 1, hd, dtype, std=std, seed=31)
    run(2, 130, 200, 1, 1, hd, dtype, -1, 0, 70, std=std, ragged=True, seed=32)
    run(1, 40, 50, 1, 1, hd, dtype, 5, 3, 0, std=std, seed=33)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_the_largest_limits_are_limits(dtype, hd):
    """left and right of 2^30 with an offset as far: causal attention, its mirror, and no key at all."""
    far = 1 << 30
    run(1, 90, 100, 1, 1, hd, dtype, -1, far, -far, seed=34)
    run(1, 90, 100, 1, 1, hd, dtype, far, -1, far, seed=35)
    run(1, 90, 100, 1, 1, hd, dtype, far, far, 0, seed=36)
    run(1, 90, 100, 1, 1, hd, dtype, far - 1, 0, far, seed=37)
