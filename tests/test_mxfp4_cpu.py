"""MXFP4 quantisers, product, linear and layers on CPU tensors, against the definition in 64 bits, and their refusals."""
import math

import pytest
import torch
import torch.nn as nn

from flex_shard_b200.ops import mxfp4 as m4
from flex_shard_b200.ops import mxfp8 as m8
from flex_shard_b200.ops.gemm import linear
from flex_shard_b200.quant import (BlockwiseMxfp4Weight, FlexShardMxfp4BlockwiseLinear,
                                   convert_to_flex_shard_mxfp4_blockwise_linear)

MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def definition(x, block):
    """(values, scale bytes) in 64 bits, element by element over the groups: nearest code, ties to the even one."""
    rows, cols = x.shape
    pad = torch.zeros(-(-rows // block) * block, cols, dtype=torch.float64)
    pad[:rows] = x.double()
    t = pad.view(-1, block, cols // 32, 32)
    out, scales = torch.zeros_like(t), torch.zeros(t.shape[0], t.shape[2], dtype=torch.uint8)
    table = torch.tensor(MAGNITUDES, dtype=torch.float64)
    for i in range(t.shape[0]):
        for j in range(t.shape[2]):
            tile = t[i, :, j]
            amax = float(tile.abs().max())
            if not math.isfinite(amax):
                scales[i, j], out[i, :, j] = 255, math.nan
                continue
            e = -127
            while amax > 6.0 * 2.0 ** e:
                e += 1
            scales[i, j] = e + 127 if amax else 0
            v = tile.abs() / 2.0 ** e
            dist = (v[..., None] - table).abs()
            near = dist.min(-1, keepdim=True).values
            even = torch.arange(8) % 2 == 0
            pick = torch.where((dist == near).sum(-1) > 1, ((dist == near) & even).int().argmax(-1), dist.argmin(-1))
            out[i, :, j] = table[pick] * torch.sign(tile) * 2.0 ** e
    return out.view(-1, cols)[:rows], scales


def hard_rows(rows, cols, seed=0):
    """Uneven rows with ties, zeros, subnormals and the largest values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
    x[0, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4) * torch.tensor([1.0, -1.0] * 16)
    if rows > 3:
        x[1, :32] = 0
        x[2, :32] = 1e-39
        x[2, 5] = 9.2e-41            # the smallest bf16 subnormal
        x[3, :32] = 3.3e38
    return x.bfloat16()


@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 96), (40, 128), (33, 160)])
def test_quantisers_match_the_definition(rows, cols):
    x = hard_rows(rows, cols)
    values, scales = definition(x, 1)
    q, s = m4.mx4_quantize_act(x)
    assert q.shape == (rows, cols // 2) and torch.equal(m8.from_blocked(s, rows, cols // 32), scales)
    assert torch.equal(m4.mx4_dequantize(q, s, torch.float32).double(), values.float().double())
    values, scales = definition(x, 32)
    q, e = m4.mx4_quantize_weight(x)
    assert torch.equal(e, scales)
    assert torch.equal(m4.mx4_dequantize(q, m8.mx_expand_scales(e, rows, cols), torch.float32).double(), values.float().double())
    q2, e2, fwd, dgrad = m4.mx4_quantize_weight_operands(x)
    assert torch.equal(q, q2) and torch.equal(e, e2)
    assert torch.equal(fwd, m8.mx_expand_scales(e, rows, cols)) and torch.equal(dgrad, m8.mx_expand_scales(e, rows, cols, True))


def test_groups_with_nan_or_infinity_are_nan():
    x = torch.ones(3, 96).bfloat16()
    x[0, 40], x[1, 70], x[2, 1] = math.inf, math.nan, -math.inf
    q, s = m4.mx4_quantize_act(x)
    v = m4.mx4_dequantize(q, s)
    bad = torch.zeros(3, 96, dtype=torch.bool)
    bad[0, 32:64], bad[1, 64:], bad[2, :32] = True, True, True
    assert torch.equal(v.isnan(), bad) and (v[~bad] == 1).all()
    _, e = m4.mx4_quantize_weight(x)
    assert e.tolist() == [[255, 255, 255]]


def test_a_code_byte_holds_the_even_column_low():
    x = torch.zeros(1, 32).bfloat16()
    x[0, 0], x[0, 1], x[0, 2] = 6.0, -0.5, 3.0
    q, s = m4.mx4_quantize_act(x)
    assert q[0, :2].tolist() == [0x97, 0x05] and int(m8.from_blocked(s, 1, 1)) == 127
    assert torch.equal(m4.mx4_to_e4m3(q).float(), m4.mx4_dequantize(q, s, torch.float32))


@pytest.mark.parametrize("T,N,K", [(128, 128, 128), (5, 128, 256), (1, 256, 128)])
def test_linear_gradients_match_their_formulas(T, N, K):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T, K, generator=g).bfloat16().requires_grad_()
    w = (torch.randn(N, K, generator=g) / K ** 0.5).bfloat16().requires_grad_()
    dy = torch.randn(T, N, generator=g).bfloat16()
    w4 = BlockwiseMxfp4Weight.from_float(w)
    y = m4.mxfp4_linear(x, w, w4.qdata, w4.scale, w4.dgrad_scale)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wv = definition(w.detach(), 32)[0]
    xv = definition(x.detach(), 1)[0]
    e8 = lambda t: m8.mx_dequantize(*m8.mx_quantize_act_ref(t)).double()  # noqa: E731
    half = 2.0 ** -8                        # one rounding to bf16, half a step

    def close(got, a, b):
        ref = a @ b
        assert ((got.double() - ref).abs() <= ref.abs() * half + (a.abs() @ b.abs()) * (a.shape[1] * 2.0 ** -24)).all()

    close(y.detach(), xv, wv.t())
    close(dx, e8(dy), wv)
    if T % 128 == 0:
        close(dw, e8(dy.t().contiguous()), e8(x.detach().t().contiguous()).t())
    else:
        close(dw, dy.double().t(), x.detach().double())


def test_layer_converter_frozen_weight_and_dispatch():
    torch.manual_seed(0)
    net = nn.Sequential(nn.Linear(128, 256, bias=False), nn.Linear(256, 128, bias=False), nn.Linear(128, 40, bias=False)).bfloat16()
    convert_to_flex_shard_mxfp4_blockwise_linear(net)
    assert [type(m) for m in net] == [FlexShardMxfp4BlockwiseLinear] * 2 + [nn.Linear]
    x = torch.randn(2, 3, 128).bfloat16().requires_grad_()
    y = net[:2](x)
    y.sum().backward()
    assert net[0].weight.grad.shape == (256, 128) and x.grad.shape == x.shape
    master = net[0].weight
    live = net[0](x).detach()
    net[0].freeze_().freeze_()
    assert isinstance(net[0].weight, BlockwiseMxfp4Weight) and not net[0].weight.requires_grad
    assert torch.equal(net[0](x).detach(), live)
    assert torch.equal(linear(x.detach(), net[0].weight), live)
    assert torch.equal(net[0].weight.dequantize().double(), definition(master.detach(), 32)[0].float().double())
    (dx,) = torch.autograd.grad(net[0](x).sum(), x)           # a frozen weight still passes gradients on
    assert dx.shape == x.shape
    with pytest.raises(ValueError, match="quantised already"):
        BlockwiseMxfp4Weight.from_float(net[0].weight)


def test_no_rows():
    x = torch.empty(0, 128).bfloat16().requires_grad_()
    w = torch.randn(128, 128).bfloat16().requires_grad_()
    w4 = BlockwiseMxfp4Weight.from_float(w)
    y = m4.mxfp4_linear(x, w, w4.qdata, w4.scale, w4.dgrad_scale)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (0, 128) and dx.shape == (0, 128) and not dw.any()


def test_second_derivatives_are_refused():
    x, w = torch.randn(4, 128).bfloat16().requires_grad_(), torch.randn(128, 128).bfloat16()
    w4 = BlockwiseMxfp4Weight.from_float(w)
    (dx,) = torch.autograd.grad(m4.mxfp4_linear(x, None, w4.qdata, w4.scale, w4.dgrad_scale).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.float().sum().backward()


def test_refusals():
    x, w = torch.zeros(4, 128).bfloat16(), torch.zeros(128, 128).bfloat16()
    w4 = BlockwiseMxfp4Weight.from_float(w)
    q, s = m4.mx4_quantize_act(x)
    with pytest.raises(ValueError, match="multiple of 32"):
        m4.mx4_quantize_act(torch.zeros(4, 40).bfloat16())
    with pytest.raises(ValueError, match="matrix"):
        m4.mx4_quantize_weight(torch.zeros(2, 4, 32).bfloat16())
    with pytest.raises(ValueError, match="floating"):
        m4.mx4_quantize_act(torch.zeros(4, 32, dtype=torch.int32))
    with pytest.raises(ValueError, match="uint8 matrix"):
        m4.gemm_mxfp4(q.int(), s, w4.qdata, w4.scale)
    with pytest.raises(ValueError, match="512 contiguous"):
        m4.gemm_mxfp4(q, s[:100], w4.qdata, w4.scale)
    with pytest.raises(ValueError, match="operands"):
        m4.gemm_mxfp4(*m4.mx4_quantize_act(torch.zeros(4, 64).bfloat16()), w4.qdata, w4.scale)
    with pytest.raises(ValueError, match="bf16 or fp32"):
        m4.gemm_mxfp4(q, s, w4.qdata, w4.scale, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="bf16 or fp32"):
        m4.mx4_dequantize(q, s, torch.float16)
    with pytest.raises(ValueError, match="bf16 inputs"):
        m4.mxfp4_linear(x.float(), None, w4.qdata, w4.scale, None)
    with pytest.raises(ValueError, match="does not match"):
        m4.mxfp4_linear(x[:, :64], None, w4.qdata, w4.scale, None)
    with pytest.raises(ValueError, match="dgrad_scale"):
        m4.mxfp4_linear(x.clone().requires_grad_(), None, w4.qdata, w4.scale, None)
    odd = BlockwiseMxfp4Weight.from_float(torch.zeros(40, 128).bfloat16())
    with pytest.raises(ValueError, match="multiples of 128"):
        m4.mxfp4_linear(x.clone().requires_grad_(), None, odd.qdata, odd.scale, odd.dgrad_scale)
    with pytest.raises(ValueError, match="multiples of 8"):
        w = torch.zeros(36, 128).bfloat16()
        w4 = BlockwiseMxfp4Weight.from_float(w)
        m4.mxfp4_linear(x, w.requires_grad_(), w4.qdata, w4.scale, w4.dgrad_scale)


@pytest.mark.parametrize("change", [lambda s: s[:-1], lambda s: s.repeat_interleave(2)[::2], lambda s: s.int(), lambda s: s.to("meta")])
def test_input_gradient_scales_are_checked(change):
    """Short, strided, wrongly typed or elsewhere: the products read them by their sizes alone."""
    x, w4 = torch.zeros(4, 128).bfloat16(), BlockwiseMxfp4Weight.from_float(torch.zeros(256, 128).bfloat16())
    with pytest.raises(ValueError, match="dgrad_scale.*contiguous uint8"):
        m4.mxfp4_linear(x.clone().requires_grad_(), None, w4.qdata, w4.scale, change(w4.dgrad_scale))
    assert m4.mxfp4_linear(x, None, w4.qdata, w4.scale, None).shape == (4, 256)
