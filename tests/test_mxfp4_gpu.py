"""MXFP4 kernels against the CPU restatement (bitwise for the quantisers) and products in 64 bits."""
import pytest
import torch

from flex_shard_b200 import ops
from flex_shard_b200.ops import mxfp4 as m4
from flex_shard_b200.ops import mxfp8 as m8
from flex_shard_b200.quant import BlockwiseMxfp4Weight, FlexShardMxfp4BlockwiseLinear

pytestmark = pytest.mark.gpu


def rows_of(rows, cols, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
    x[0, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4) * torch.tensor([1.0, -1.0] * 16)
    if rows > 4:
        x[1, :32] = 0
        x[2, :32] = 1e-39
        x[3, :32] = 3.3e38
        x[4, 7] = float("nan")
        x[4, 40 % cols] = float("inf")
    return x.bfloat16()


@pytest.mark.parametrize("rows,cols,pad", [(1, 32, 0), (7, 96, 0), (129, 160, 0), (300, 4128, 0), (64, 256, 8), (33, 64, 3), (257, 2048, 1), (2500, 4128, 0)])
def test_quantisers_match_the_restatement_bitwise(rows, cols, pad):
    """Odd sizes, groups and rows that end inside a scale block, row strides and bases off the 16-byte grid."""
    x = rows_of(rows, cols + 32, 3)[:, pad:pad + cols]
    xg = rows_of(rows, cols + 32, 3).cuda()[:, pad:pad + cols]
    q, s = m4.mx4_quantize_act(xg)
    q_ref, s_ref = m4.mx4_quantize_act(x)
    assert torch.equal(q.cpu(), q_ref) and torch.equal(s.cpu(), s_ref)          # padding bytes included
    for dt in (torch.bfloat16, torch.float32):
        torch.testing.assert_close(m4.mx4_dequantize(q, s, dt).cpu(), m4.mx4_dequantize(q_ref, s_ref, dt), rtol=0, atol=0, equal_nan=True)
    assert torch.equal(m4.mx4_to_e4m3(q).cpu().view(torch.uint8), m4.mx4_to_e4m3(q_ref).view(torch.uint8))
    got, ref = m4.mx4_quantize_weight_operands(xg), m4.mx4_quantize_weight_operands(x)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, ref))
    q, e = m4.mx4_quantize_weight(xg)
    assert torch.equal(q.cpu(), ref[0]) and torch.equal(e.cpu(), ref[1])


def operand(rows, K, seed):
    g = torch.Generator().manual_seed(seed)
    q, s = m4.mx4_quantize_act_ref((torch.randn(rows, K, generator=g) * (0.1 + torch.rand(rows, 1, generator=g))).bfloat16())
    return q.cuda(), s.cuda(), m4.mx4_dequantize(q, s, torch.float32).double().cuda()


def check_product(y, a, b):
    """Products of two 4-bit values and powers of two are exact; a sum of K of them is good to K 2^-24 of the magnitudes' sum,
    and bf16 rounds by half a step, 2^-8."""
    ref = a @ b.t()
    bound = (a.abs() @ b.abs().t()) * (a.shape[1] * 2.0 ** -24) + ref.abs() * (2.0 ** -8 if y.dtype == torch.bfloat16 else 0)
    assert y.shape == ref.shape and ((y.double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("M,N,K", [
    (1, 128, 256), (1, 1, 32), (1, 4096, 4096), (3, 130, 96), (16, 256, 160), (17, 384, 1024), (32, 100, 2080), (48, 1000, 512),
    (64, 129, 4096), (65, 128, 128), (128, 512, 1152), (129, 300, 640), (257, 1000, 800), (777, 1290, 416), (1024, 2048, 256), (513, 257, 32), (600, 3000, 1056),
    (2305, 2440, 288), (4104, 1560, 384), (1300, 9000, 4096),
    (100, 300, 14400), (130, 260, 7200), (33, 70, 9248), (20, 1111, 5984)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_product(M, N, K, dt):
    aq, sa, a = operand(M, K, 1)
    bq, sb, b = operand(N, K, 2)
    y = m4.gemm_mxfp4(aq, sa, bq, sb, out_dtype=dt)
    ops.check_status()
    check_product(y, a, b)


def test_product_of_strided_codes_and_nan_groups():
    M, N, K = 70, 200, 512
    aq, sa, a = operand(M, K, 3)
    bq, sb, b = operand(N, K, 4)
    wide = torch.zeros(N, 3 * K // 2, dtype=torch.uint8, device="cuda")
    for at in (K // 2, 8):                               # a 16-byte-aligned column offset, and one that is not
        wide[:, at:at + K // 2] = bq
        check_product(m4.gemm_mxfp4(aq, sa, wide[:, at:at + K // 2], sb), a, b)
    x = torch.ones(M, K).bfloat16()
    x[5, 300] = float("nan")
    xq, sx = m4.mx4_quantize_act(x.cuda())
    y = m4.gemm_mxfp4(xq, sx, bq, sb)
    bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[5] = True
    assert torch.equal(y.isnan(), bad)
    ops.check_status()


@pytest.mark.parametrize("T,N,K,pad", [
    (1, 128, 32, 0), (1, 1, 64, 0), (2, 300, 2080, 8), (5, 1000, 4128, 3), (16, 200, 1056, 0), (9, 4096, 14336, 0), (16, 131, 288, 1),
    (3, 257, 40000, 0), (1, 6144, 4096, 0), (12, 40, 106496, 0), (1, 64, 110016, 0), (17, 300, 2080, 0), (90, 513, 800, 5)])
def test_scoring_with_a_frozen_weight(T, N, K, pad):
    """The quantiser and the product behind one call, inside one kernel for few rows: sums of K products in parts, in fp32."""
    g = torch.Generator(device="cuda").manual_seed(6)
    base = torch.randn(T, K + pad, generator=g, device="cuda").bfloat16()
    x = base[:, pad:]
    bq, sb, b = operand(N, K, 7)
    y = m4.mxfp4_linear(x, None, bq, sb, None)
    ops.check_status()
    check_product(y, m4.mx4_dequantize(*m4.mx4_quantize_act(x), torch.float32).double(), b)
    assert torch.equal(y, m4.mxfp4_linear(x, None, bq, sb, None))
    assert torch.equal(m4.mxfp4_linear(x[None], None, bq, sb, None), y[None])
    x[T - 1, K - 1] = float("inf")
    y = m4.mxfp4_linear(x, None, bq, sb, None)
    assert y[T - 1].isnan().all() and not y[:T - 1].isnan().any()


@pytest.mark.parametrize("T,N,K", [(1, 256, 128), (100, 128, 384), (384, 512, 256), (256, 1152, 640)])
def test_linear_and_its_gradients(T, N, K):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(T, K, generator=g).bfloat16().cuda().requires_grad_()
    w = (torch.randn(N, K, generator=g) / K ** 0.5).bfloat16().cuda().requires_grad_()
    dy = torch.randn(T, N, generator=g).bfloat16().cuda()
    w4 = BlockwiseMxfp4Weight.from_float(w)
    y = m4.mxfp4_linear(x, w, w4.qdata, w4.scale, w4.dgrad_scale)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ops.check_status()
    wv = w4.dequantize().double()
    xv = m4.mx4_dequantize(*m4.mx4_quantize_act(x), torch.float32).double()
    e8 = lambda t: m8.mx_dequantize(*(s.cuda() for s in m8.mx_quantize_act_ref(t.detach().cpu()))).double()  # noqa: E731
    check_product(y, xv, wv)
    check_product(dx, e8(dy), wv.t())
    if T % 128 == 0:
        check_product(dw, e8(dy.t().contiguous()), e8(x.t().contiguous()))
    else:
        check_product(dw, dy.double().t(), x.detach().double().t())


def test_sizes_that_pass_32_bits():
    """Codes, inputs and outputs whose last rows lie past 2^31 elements."""
    T, K, N = 1_049_700, 2048, 2064
    base = torch.randn(64, K, device="cuda").bfloat16()
    x = base.repeat(T // 64 + 1, 1)[:T]
    same = torch.arange(T - 100, T, device="cuda") % 64     # rows of the base that the last rows repeat
    q, s = m4.mx4_quantize_act(x)
    q_ref, s_ref = m4.mx4_quantize_act(base)
    assert torch.equal(q[-100:], q_ref[same])
    bq, sb, b = operand(N, K, 8)
    y = m4.gemm_mxfp4(q, s, bq, sb)
    ops.check_status()
    check_product(y[-100:], m4.mx4_dequantize(q_ref, s_ref, torch.float32).double()[same], b)
    del y
    assert torch.equal(m4.mx4_dequantize(q, s)[-100:], m4.mx4_dequantize(q_ref, s_ref)[same])


def test_a_single_row_of_any_stride():
    K, N = 256, 40
    bq, sb, b = operand(N, K, 9)
    aq, sa, a = operand(1, K, 10)
    odd = torch.zeros(K // 2, 3, dtype=torch.uint8, device="cuda")
    odd[:, 1] = aq[0]
    row = odd[:, 1:2].t()                                   # [1, K / 2] with strides (1, 3)
    check_product(m4.gemm_mxfp4(row, sa, bq, sb), a, b)
    check_product(m4.gemm_mxfp4(aq.as_strided((1, K // 2), (7, 1)), sa, bq, sb), a, b)
    assert torch.equal(m4.mx4_dequantize(row, sa), m4.mx4_dequantize(aq, sa))


@pytest.mark.parametrize("grad_bucket", [False, True])
def test_sharded_layers_train_like_unsharded_ones(grad_bucket):
    """The gradients of a sharded stack (written into the bucket where it offers its rows) and of the plain one; an fp32 bucket
    takes them unrounded, the plain weight in bf16."""
    from flex_shard_b200 import BucketSpec, MixedPrecisionPolicy, flex_shard
    from flex_shard_b200.placements.shard import shard_placement_fn

    def net():
        torch.manual_seed(0)
        m = torch.nn.Sequential(FlexShardMxfp4BlockwiseLinear(256, 384, device="cuda"), FlexShardMxfp4BlockwiseLinear(384, 128, device="cuda"))
        for p in m.parameters():
            torch.nn.init.normal_(p, std=0.05)
        return m

    x, dy = torch.randn(200, 256, device="cuda").bfloat16(), torch.randn(200, 128, device="cuda").bfloat16()
    plain, sharded = net(), net()
    flex_shard(sharded, [BucketSpec(["*"], mp_policy=MixedPrecisionPolicy(param_dtype=torch.bfloat16, reduce_dtype=torch.float32),
                                    placement_fn=shard_placement_fn(0, grad_bucket=grad_bucket))])
    y, z = plain(x), sharded(x)
    assert torch.equal(y, z)
    y.backward(dy)
    z.backward(dy)
    ops.check_status()
    for a, b in zip(plain.parameters(), sharded.parameters()):
        ga, gb = a.grad.double(), b.grad.double().view(a.shape)
        assert gb.any() and ((ga - gb).abs() <= gb.abs() * 2.0 ** -7).all()     # one rounding to bf16 on either side


def test_layer_trains_and_scores_in_a_captured_graph():
    torch.manual_seed(0)
    layer = FlexShardMxfp4BlockwiseLinear(256, 512, device="cuda")
    torch.nn.init.normal_(layer.weight, std=0.05)
    x = torch.randn(4, 33, 256, device="cuda").bfloat16()
    y = layer(x)
    y.float().square().mean().backward()
    assert layer.weight.grad.shape == (512, 256) and layer.weight.grad.isfinite().all()
    layer.freeze_()
    layer.weight.grad = None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        assert torch.equal(layer(x), y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            z = layer(x)
    torch.cuda.current_stream().wait_stream(side)
    fresh = torch.randn_like(x)
    x.copy_(fresh)
    graph.replay()
    graph.replay()
    with torch.no_grad():
        assert torch.equal(z, layer(fresh))
    ops.check_status()


@pytest.mark.parametrize("rows,cols", [(1, 32), (33, 96), (128, 128), (300, 4128), (4100, 160)])
def test_expanded_tile_exponents_match_the_restatement(rows, cols):
    e = torch.randint(0, 255, (-(-rows // 32), cols // 32), dtype=torch.uint8)
    for transpose in (False, True):
        assert torch.equal(m8.mx_expand_scales(e.cuda(), rows, cols, transpose).cpu(), m8.mx_expand_scales(e, rows, cols, transpose))


@pytest.mark.parametrize("T", [1, 5, 127, 128, 384])
@pytest.mark.parametrize("layout", ["plain", "strided codes", "codes off a word", "scales off a vector", "strided input"])
def test_gradients_are_those_of_the_separate_operators(T, layout):
    """The joint entries against the public quantisers and products that they run, bit for bit."""
    from flex_shard_b200.ops.mxfp8 import gemm_mxfp8, mx_quantize_act, mx_quantize_rows

    N, K = 256, 384
    g = torch.Generator("cuda").manual_seed(T)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    x, w, dy = rand(T, K), rand(N, K), rand(T, N)
    w4 = BlockwiseMxfp4Weight.from_float(w)
    wq, sd = w4.qdata, w4.dgrad_scale
    if layout == "strided codes":
        wq = torch.cat([wq, wq], 1)[:, : K // 2]
    elif layout == "codes off a word":
        wq = torch.cat([wq.flatten()[:1], wq.flatten()])[1:].view(N, K // 2)
    elif layout == "scales off a vector":
        sd = torch.cat([sd[:1], sd])[1:]
    elif layout == "strided input":
        x = torch.cat([x, x], 1)[:, :K]
    xg, wg = x.detach().requires_grad_(), w.requires_grad_()
    for dtype in (torch.bfloat16, torch.float32):
        wg.grad_dtype = dtype
        y = m4.mxfp4_linear(xg, wg, wq, w4.scale, sd)
        dx, dw = torch.autograd.grad(y, (xg, wg), dy)
        want = gemm_mxfp8(*mx_quantize_act(dy), m4.mx4_to_e4m3(w4.qdata), w4.dgrad_scale, b_t=True)
        assert torch.equal(dx, want)
        if T % 128 == 0:
            want = gemm_mxfp8(*mx_quantize_rows(dy), *mx_quantize_rows(x), a_t=True, b_t=True, out_dtype=dtype)
            assert dw.dtype == dtype and torch.equal(dw, want)
