"""Token log probabilities where the logits are large against the temperature: kernels against the definition in 64 bits."""
import pytest
import torch

from tests import logprobs_far_common as far
from tests.logprobs_far_common import BF, FP, HF

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [0.1, 0.01, 1e-3, 1e-4, 1e-5, 1e-6, 1e-7, 1e-8, 1e-12, 1e-30, 1e4, 1e30])
@pytest.mark.parametrize("V,T,dtype", [(1000, 5, FP), (32000, 3, FP), (32000, 3, BF), (5001, 700, BF), (128256, 2, BF), (4099, 7, HF), (3, 4, FP)])
def test_low_temperatures(V, T, dtype, temperature):
    far.low_temperatures(V, T, dtype, temperature, "cuda")


@pytest.mark.parametrize("V,dtype,offset", [(1000, FP, o) for o in (1e3, 3e4, -3e4, 1e6, 1e8, -1e8, 1e12, -1e30)]
                         + [(20000, BF, 1e3), (20000, BF, 3e4), (9001, HF, 3e4), (128256, FP, 1e6), (50, FP, 1e6)])
def test_common_offsets(V, dtype, offset):
    far.common_offsets(V, dtype, offset, "cuda")


@pytest.mark.parametrize("dtype,value", [(FP, 1e8), (FP, 3e4), (FP, -1e9), (FP, 123.456), (FP, 3e38), (BF, 3e4), (BF, -1e30), (HF, 6e4)])
def test_one_token(dtype, value):
    far.one_token(dtype, value, "cuda")


@pytest.mark.parametrize("V,dtype,value", [(1000, FP, -1e9), (32000, FP, -1e12), (4000, BF, -1e9), (70000, FP, 1e9), (1000, FP, -1e30),
                                           (1000, HF, -65504.0), (40000, BF, 1e4)])
def test_equal_rows(V, dtype, value):
    far.equal_rows(V, dtype, value, "cuda")


@pytest.mark.parametrize("V,dtype,mask", [(v, d, m) for v in (1003, 33000) for d, m in ((FP, -1e4), (FP, -1e9), (FP, -1e30), (BF, -1e9),
                                                                                        (BF, -1e30), (HF, -65504.0), (HF, -1e4))])
def test_finite_masks(V, dtype, mask):
    far.finite_masks(V, dtype, mask, "cuda")
