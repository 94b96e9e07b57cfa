"""Token log probabilities where the logits are large against the temperature: CPU tensors against the definition in 64 bits."""
import pytest
import torch

from tests import logprobs_far_common as far
from tests.logprobs_far_common import BF, FP, HF


@pytest.mark.parametrize("temperature", [0.1, 1e-3, 1e-6, 1e-12, 1e-30, 1e30])
@pytest.mark.parametrize("V,dtype", [(1000, FP), (2000, BF), (3, HF)])
def test_low_temperatures(V, dtype, temperature):
    far.low_temperatures(V, 5, dtype, temperature, "cpu")


@pytest.mark.parametrize("dtype,offset", [(FP, 3e4), (FP, 1e6), (FP, -1e8), (FP, 1e30), (BF, 3e4), (HF, 3e4)])
def test_common_offsets(dtype, offset):
    far.common_offsets(1000, dtype, offset, "cpu")


@pytest.mark.parametrize("dtype,value", [(FP, 1e8), (FP, 123.456), (BF, -1e30), (HF, 6e4)])
def test_one_token(dtype, value):
    far.one_token(dtype, value, "cpu")


@pytest.mark.parametrize("dtype,value", [(FP, -1e9), (BF, -1e12), (HF, -65504.0)])
def test_equal_rows(dtype, value):
    far.equal_rows(1000, dtype, value, "cpu")


@pytest.mark.parametrize("dtype,mask", [(FP, -1e9), (BF, -1e30), (HF, -65504.0)])
def test_finite_masks(dtype, mask):
    far.finite_masks(1003, dtype, mask, "cpu")
