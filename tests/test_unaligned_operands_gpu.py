"""Dense operands and gradients that start anywhere in memory: the results of aligned copies, bit for bit."""
import pytest
import torch

from flex_shard_b200 import ops
from flex_shard_b200.ops import attention
from flex_shard_b200.ops import elementwise as ew
from flex_shard_b200.ops import fp8, moe, mxfp4, mxfp8
from flex_shard_b200.ops.attention import qkv_attention
from flex_shard_b200.ops.gemm import linear
from flex_shard_b200.quant import BlockwiseMxfp4Weight

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


@pytest.mark.parametrize("T,K", [(1, 128), (7, 256), (129, 384)])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (2, 0), (4, 0), (6, 0), (0, 1), (3, 2), (0, 4), (4, 4), (8, 8), (1, 7)])
def test_mxfp8_quantiser(T, K, offset, pad):
    """Bases and row strides of every alignment."""
    x = rand(T, K + pad)
    q, s = mxfp8.mx_quantize_act(off(x, offset)[:, :K])
    ops.check_status()
    q_ref, s_ref = mxfp8.mx_quantize_act_ref(x[:, :K].cpu())
    assert torch.equal(q.cpu().view(torch.uint8), q_ref.view(torch.uint8))
    assert torch.equal(mxfp8.from_blocked(s, T, K // 32).cpu(), mxfp8.from_blocked(s_ref, T, K // 32))


@pytest.mark.parametrize("T", [1, 100, 128])
@pytest.mark.parametrize("offset", [1, 4, 7])
def test_block_scaled_linears(T, offset):
    """Inputs and gradients off a boundary; 128 rows take the 8-bit weight gradient, fewer the bf16 one."""
    x, w, dy = rand(T, 256), rand(384, 256, seed=1), rand(T, 384, seed=2)
    w4 = BlockwiseMxfp4Weight.from_float(w)
    q8, e8 = mxfp8.mx_quantize_weight(w)
    scales = [mxfp8.mx_expand_scales(e8, 384, 256, transpose) for transpose in (False, True)]
    for f in (lambda x, w: mxfp4.mxfp4_linear(x, w, w4.qdata, w4.scale, w4.dgrad_scale), lambda x, w: mxfp8.mxfp8_linear(x, w, q8, *scales)):

        def run(x, dy):
            a, b = x.requires_grad_(), w.detach().requires_grad_()
            y = f(a, b)
            return y, *torch.autograd.grad(y, (a, b), dy)

        want, got = run(x.clone(), dy), run(off(x, offset), off(dy, offset))
        ops.check_status()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_gradient_behind_a_concatenation():
    """A dense gradient that starts one element into its memory, as an ordinary program makes it."""
    x, w = rand(8, 128).requires_grad_(), rand(128, 128, seed=1)
    w4 = BlockwiseMxfp4Weight.from_float(w)
    weight = rand(8 * 128 + 1, seed=2)
    y = linear(x, torch.nn.Parameter(w4, requires_grad=False))
    (dx,) = torch.autograd.grad((torch.cat([torch.ones(1, device="cuda").bfloat16(), y.flatten()]) * weight).sum(), x)
    y = linear(x, torch.nn.Parameter(w4, requires_grad=False))
    (want,) = torch.autograd.grad(y, x, weight[1:].clone().view(8, 128))
    assert torch.equal(dx, want)


@pytest.mark.parametrize("T,K", [(1, 128), (7, 256), (129, 384)])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (2, 0), (4, 0), (6, 0), (0, 1), (3, 2), (0, 4), (4, 4), (8, 8), (1, 7)])
def test_fp8_quantisers(T, K, offset, pad):
    """Bases and row strides of every alignment give the bits of a dense, aligned copy; a weight also with columns that end
    inside a vector."""
    x = rand(T, K + pad)
    got, want = fp8.quantize_act(off(x, offset)[:, :K]), fp8.quantize_act(x[:, :K].clone())
    ops.check_status()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    for cols in (K, K - 5):
        got = fp8.quantize_blockwise(off(x, offset)[:, :cols])
        q, s = fp8.quantize_blockwise_ref(x[:, :cols].cpu())
        assert torch.equal(got[0].cpu().view(torch.uint8), q.view(torch.uint8)) and torch.equal(got[1].cpu(), s)


@pytest.mark.parametrize("offset", [1, 4, 7])
def test_fp8_linear(offset):
    x, w, dy = rand(100, 256), rand(384, 256, seed=1), rand(100, 384, seed=2)
    q, s = fp8.quantize_blockwise(w)

    def run(x, dy):
        a, b = x.requires_grad_(), w.detach().requires_grad_()
        y = fp8.fp8_linear(a, b, q, s)
        return y, *torch.autograd.grad(y, (a, b), dy)

    want, got = run(x.clone(), dy), run(off(x, offset), off(dy, offset))
    ops.check_status()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def same(f, inputs, gradients, offset):
    """Outputs and gradients of ``f`` from aligned inputs and from those that start ``offset`` elements into their memory."""
    results = []
    for at in (0, offset):
        xs = [off(x, at).requires_grad_() for x in inputs]
        ys = f(*xs)
        ys = ys if isinstance(ys, tuple) else (ys,)
        results.append([*ys, *torch.autograd.grad(ys, xs, [off(g, at) for g in gradients])])
    ops.check_status()
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("offset", [1, 4])
def test_norms_and_activation(offset):
    x, r, w = rand(37, 256), rand(37, 256, seed=1), rand(256, seed=2)
    same(lambda x, w: ew.rmsnorm(x, w), (x, w), (r,), offset)
    same(lambda x, r, w: ew.add_rmsnorm(x, r, w), (x, r, w), (rand(37, 256, seed=3), rand(37, 256, seed=4)), offset)
    same(ew.swiglu, (x,), (rand(37, 128, seed=3),), offset)


@pytest.mark.parametrize("offset", [1, 4])
def test_attention(offset):
    """The input is rotated in place on the GPU, so every run has its own."""
    B, S = 1, 128
    table = ew.rope_table(S, 128, 10000.0, "cuda")
    o = qkv_attention(off(rand(B, S, 4 * 128), 0), table, 2, 1)
    p = qkv_attention(off(rand(B, S, 4 * 128), offset), table, 2, 1)
    assert torch.equal(o, p)
    attention.set_deterministic(True)           # otherwise the query gradient is added up in any order
    try:
        results = []
        for at in (0, offset):
            x = rand(B, S, 4 * 128).requires_grad_()
            y = qkv_attention(x * 1, table, 2, 1)
            results.append(torch.autograd.grad(y, x, off(rand(B, S, 2 * 128, seed=1), at))[0])
        ops.check_status()
    finally:
        attention.set_deterministic(None)
    assert torch.equal(*results)


@pytest.mark.parametrize("offset", [1, 4])
def test_experts(offset):
    T, k, E, D, F = 100, 2, 4, 128, 256
    plan = moe.plan_routes(torch.stack([torch.randperm(E, device="cuda")[:k] for _ in range(T)]), E)
    same(lambda x: moe.moe_dispatch(x, plan), (rand(T, D),), (rand(plan.max_rows, D, seed=1),), offset)
    rows, w = moe.moe_dispatch(rand(T, D), plan), torch.rand(T, k, device="cuda")
    same(lambda r: moe.moe_combine(r, w, plan), (rows,), (rand(T, D, seed=2),), offset)
    weight = rand(E, F, D, seed=3)
    live = (plan.src >= 0)[:, None]
    x = rows.detach().requires_grad_()
    dy = rand(plan.max_rows, F, seed=4) * live
    got = [torch.autograd.grad(moe.grouped_linear(x, weight, plan), x, off(dy, at))[0] * live for at in (0, offset)]
    ops.check_status()
    assert torch.equal(*got)
