"""Products that contract over the rows of both operands, for any number of rows (weight gradients of any token count)."""
import pytest
import torch

from flex_shard_b200 import ops
from flex_shard_b200.ops.gemm import linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(128, 256, 1), (264, 320, 77), (64, 8, 7), (2048, 1024, 503), (1024, 2048, 1001), (256, 256, 65)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_any_number_of_rows(M, N, K, dt):
    """bf16 products are exact in fp32; sums of K of them are good to K 2^-24 of the magnitudes' sum, bf16 rounds by 2^-8."""
    g = torch.Generator(device="cuda").manual_seed(0)
    a = torch.randn(K, M, generator=g, device="cuda").bfloat16()
    b = torch.randn(K, N, generator=g, device="cuda").bfloat16()
    y = ops.gemm(a, b, a_t=True, b_t=True, out_dtype=dt).double()
    ops.check_status()
    ref, size = a.double().t() @ b.double(), a.double().abs().t() @ b.double().abs()
    assert ((y - ref).abs() <= size * (K * 2.0 ** -24) + ref.abs() * (2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -24)).all()


def test_linear_trains_on_an_odd_number_of_tokens():
    x = torch.randn(3, 7, 64, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(128, 64, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(3, 7, 128, device="cuda").bfloat16()
    (dw,) = torch.autograd.grad(linear(x, w), w, dy)
    ref = dy.double().reshape(-1, 128).t() @ x.detach().double().reshape(-1, 64)
    size = dy.double().abs().reshape(-1, 128).t() @ x.detach().double().abs().reshape(-1, 64)
    assert ((dw.double() - ref).abs() <= size * (21 * 2.0 ** -24) + ref.abs() * 2.0 ** -8).all()
    for bad in ((4, 12), (12, 4)):
        with pytest.raises(ValueError, match="multiple of 8"):
            ops.gemm(torch.zeros(8, bad[0], device="cuda").bfloat16(), torch.zeros(8, bad[1], device="cuda").bfloat16(), a_t=True, b_t=True)
