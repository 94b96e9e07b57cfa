"""Dense operands and gradients that start anywhere in memory: the results of aligned copies, bit for bit."""
import pytest
import torch

from flex_shard_b200 import ops
from flex_shard_b200.ops.gemm import linear

pytestmark = pytest.mark.gpu


def off(t, offset):
    """A dense copy of ``t`` that starts ``offset`` elements into its memory."""
    base = torch.empty(t.numel() + offset, dtype=t.dtype, device=t.device)
    base[offset:] = t.detach().reshape(-1)
    return base[offset:].view(t.shape)


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").bfloat16()


@pytest.mark.parametrize("offset", [1, 2, 4, 6])
def test_bf16_linear(offset):
    x, w, dy = rand(100, 128), rand(256, 128, seed=1), rand(100, 256, seed=2)

    def run(x, w, dy):
        x, w = x.requires_grad_(), w.requires_grad_()
        y = linear(x, w)
        return y, *torch.autograd.grad(y, (x, w), dy)

    want = run(x.clone(), w.clone(), dy)
    got = run(off(x, offset), off(w, offset), off(dy, offset))
    ops.check_status()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
