"""The shapes of test_int8_plans_gpu.py take the kernels they stand for, and together every one that any shape takes."""

import random

import pytest

from dmf_b200 import _lib
from tests.int8_plans import PLANS


def test_shapes_take_the_kernels_they_stand_for():
    for name, shapes in PLANS.items():
        for M, K, N in shapes:
            assert _lib.int8_linear_kernel_name(M, N, K) == name, (M, K, N)


def test_no_shape_takes_a_kernel_that_is_not_covered():
    rng = random.Random(0)
    spread = lambda lo, hi: round(lo * (hi / lo) ** rng.random())
    for _ in range(50000):
        M, K, N = spread(1, 1 << 17), spread(1, 131071), spread(1, 1 << 15)
        assert _lib.int8_linear_kernel_name(M, N, K) in PLANS, (M, K, N)


def test_refusals():
    for M, N, K in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), (1, 2 ** 30 + 1, 1)):
        with pytest.raises(_lib.DmfAttnError):
            _lib.int8_linear_kernel_name(M, N, K)
