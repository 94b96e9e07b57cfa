"""SwiGLU of rows that are not dense: values and gradients of a dense copy, bit for bit."""
import pytest
import torch

from flex_shard_b200.ops import elementwise as ew

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cut", [lambda w: w[:, 16:16 + 256], lambda w: w[::2, :256], lambda w: w.t()[:256].t()])
def test_strided_rows(cut):
    wide = torch.randn(64, 512, generator=torch.Generator("cuda").manual_seed(0), device="cuda").bfloat16()
    dh = None
    results = []
    for x in (cut(wide).detach(), cut(wide).clone(memory_format=torch.contiguous_format)):
        x = x.requires_grad_()
        h = ew.swiglu(x)
        dh = torch.randn_like(h) if dh is None else dh
        results.append((h, torch.autograd.grad(h, x, dh)[0]))
    (h, dx), (h2, dx2) = results
    assert torch.equal(h, h2) and torch.equal(dx, dx2)
