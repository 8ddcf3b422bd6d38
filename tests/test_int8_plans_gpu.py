import pytest
import torch

from tests.int8_plans import PLANS
from tests.test_int8_gpu import BF16, F32, FP16, _check_linear, _pitched, _random8, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [s for shapes in PLANS.values() for s in shapes], ids=str)
@pytest.mark.parametrize("out_dtype", [BF16, FP16, F32])
def test_every_cut_of_a_product(shape, out_dtype):
    M, K, N = shape
    x, w = _pitched(_random8(M, K)), _pitched(_random8(N, K, seed=1))
    _check_linear(x, w, _randn(N), out_dtype)
