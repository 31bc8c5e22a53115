"""Attention with its gradient on values far from 1 (n3d_attention_forward, n3d_attention_backward), against 64
bits within the bounds derived in test_train_attention.py."""

import pytest

from test_train_attention import run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("std", [1e-20, 1e-30])
def test_tiny_queries_and_keys_attend_evenly(dtype, hd, std):
    run(1, 130, 200, 2, 1, hd, dtype, std=std, seed=31)
    run(2, 130, 200, 1, 1, hd, dtype, -1, 0, 70, std=std, ragged=True, seed=32)
    run(1, 40, 50, 1, 1, hd, dtype, 5, 3, 0, std=std, seed=33)
