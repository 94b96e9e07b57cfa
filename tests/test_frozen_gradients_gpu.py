"""Gradients through frozen 4-bit matrices of any size, on the GPU."""
import pytest

from flex_shard_b200 import ops
from tests.test_frozen_gradients_cpu import SIZES, check_input_gradient

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,N,K", SIZES + [(300, 2112, 1056), (128, 520, 4128)])
def test_matrices_of_any_size_pass_gradients_on(T, N, K):
    check_input_gradient(T, N, K, "cuda")
    ops.check_status()
