"""Token log probability kernels against the definition in 64 bits."""
import math

import pytest
import torch

from flex_shard_b200 import ops
from flex_shard_b200.ops.logprobs import token_logprobs
from tests.logprobs_common import HALF_STEP, SMALLEST, definition, gradient, value_tolerance

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def check(x, t, temperature=1.0, k=0, grads=True, seed=1):
    """Values, alternatives (exactly) and gradients of CUDA rows ``x``, which keep their strides."""
    T, V = x.shape
    before = x.detach().clone()
    x = x.detach().requires_grad_(grads)
    out = token_logprobs(x, t, temperature=temperature, top_k=k)
    ops.check_status()
    _, ref = definition(before, t, temperature, k)
    tol = value_tolerance(before, temperature)
    # The result is an fp32 number: a masked token's -3.39e38 / 0.9 is minus infinity there. Values of that size carry the
    # relative roundings of the difference, the reciprocal, the product and the last subtraction: 4 times 2^-24.
    for name in ("logprob", "entropy", "top_logprob"):
        torch.testing.assert_close(getattr(out, name), ref[name].float(), rtol=2.0 ** -22, atol=tol * (1 + math.log(V)),
                                   equal_nan=True, msg=lambda m: f"{name}: {m}")  # noqa: B023
    assert torch.equal(out.top_index, ref["top_index"])
    if not grads:
        return
    g = torch.Generator(device="cuda").manual_seed(seed)
    gl, gh, gt = (torch.randn(n, generator=g, device="cuda") for n in ((T,), (T,), (T, k)))
    (dx,) = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, [gl, gh, gt])
    want, size = gradient(before, t, temperature, k, gl, gh, gt)
    assert dx.shape == x.shape and dx.dtype == x.dtype
    off = (dx.double() - want).abs()
    # A probability below 2^-126 (log probability below -87.4) counts as 0: p (G + h (log p + H)), which falls with p there, is
    # then missing, at most 2^-126 (|G| + |h| (88 + ln V)).
    lost = 2.0 ** -126 * (gl.abs() + gt.abs().sum(1) + gh.abs() * (88 + math.log(V)))[:, None] / temperature
    bound = want.abs() * HALF_STEP[x.dtype] + size * 8 * tol * (1 + math.log(V)) + SMALLEST[x.dtype] + lost
    good = want.isfinite().all(1)
    assert (off <= bound)[good].all(), float((off - bound)[good].max())
    assert dx[~good].isnan().all()


def rows(T, V, dtype, seed=0, ld=None, at=0):
    """[T, V] rows with stride ``ld`` that start ``at`` elements into their memory."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = V if ld is None else ld
    base = (torch.randn(T * ld + at, generator=g, device="cuda") * 3).to(dtype)
    return base[at:].view(T, ld)[:, :V], torch.randint(0, V, (T,), generator=g, device="cuda")


@pytest.mark.parametrize("T,V,k,dtype", [
    (1, 1, 1, BF), (2, 2, 2, FP), (3, 7, 5, HF), (5, 31, 31, BF), (4, 33, 32, FP), (1, 100, 20, BF), (17, 511, 8, HF),
    (3, 1000, 32, BF), (7, 4097, 20, BF), (6, 4100, 9, FP), (300, 8192, 5, BF), (2, 32003, 32, HF), (5, 50021, 16, FP),
    (1, 128256, 20, BF), (40, 128256, 8, BF), (3, 160001, 32, FP), (1000, 333, 4, BF), (2, 300007, 20, BF)])
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_values_alternatives_and_gradient(T, V, k, dtype, temperature):
    x, t = rows(T, V, dtype)
    check(x, t, temperature, k)
    check(x, t, temperature, 0, grads=False)


@pytest.mark.parametrize("V,ld,at,dtype", [(1000, 1008, 0, BF), (1001, 1008, 0, BF), (1001, 1001, 3, BF), (999, 1003, 1, HF),
                                           (514, 517, 2, FP), (50000, 50021, 5, BF), (4096, 4097, 0, FP)])
def test_strided_and_unaligned_rows(V, ld, at, dtype):
    x, t = rows(9, V, dtype, 2, ld, at)
    check(x, t, 1.0, 6)
    wide = rows(9, 2 * V, dtype, 3)[0][:, ::2]              # columns that are not dense
    check(wide, t, 1.0, 6)


def test_masks():
    """Masked tokens (minus infinity, or the type's lowest value), rows with few or no tokens left, infinities and NaN."""
    for dtype in (BF, HF, FP):
        V = 9001
        for lowest in (-math.inf, torch.finfo(dtype).min):
            x, t = rows(8, V, dtype, 4)
            x[1, ::2] = lowest
            x[2, 5:] = lowest                              # fewer tokens left than alternatives asked for
            x[3, :-3] = lowest
            x[4, :] = lowest
            x[5, 100:8000] = lowest
            x[6, :] = lowest
            x[6, 4000] = 2.0
            t = torch.tensor([5, 1, 2, V - 1, 7, 3, 4000, 0], device="cuda")
            t[7] = -100
            check(x, t, 0.9, 20)
            check(x, t, 1.0, 1)
        x, t = rows(5, V, dtype, 5)
        x[0, 77], x[1, 8000], x[2, 3], x[2, 9] = math.inf, math.nan, math.inf, math.inf
        x[3, 10], x[3, 11], x[3, 12] = math.nan, -math.nan, math.inf
        check(x, t, 1.0, 12)


@pytest.mark.parametrize("k", [1, 7, 32])
def test_equal_and_clustered_logits(k):
    """Rows of one value, few values, large values packed where one thread or one warp reads them, and sorted rows."""
    V = 40000
    x = torch.zeros(12, V, device="cuda", dtype=BF)
    x[1, ::3] = 1.0
    x[2, 20000:] = -1.0
    x[3] = torch.linspace(-20, 20, V, device="cuda")
    x[4] = torch.linspace(20, -20, V, device="cuda")
    x[5, ::4096] = 5.0
    x[6, 8::4096] = torch.linspace(5, 9, len(range(8, V, 4096)), device="cuda").to(BF)
    for j in range(8):
        x[7, 16 + j::2048] = 3.0 + j
        x[8, 24 + j::8192] = 4.0
    x[9, 1000:1256] = 7.0
    x[10] = torch.arange(V, device="cuda") % 512
    x[11, -1] = 1.0
    t = torch.arange(12, device="cuda") * 3000
    check(x, t, 1.0, k)
    check(x.float() + torch.arange(V, device="cuda") * 1e-5, t, 1.0, k)


def test_ignored_rows_and_targets_outside_the_vocabulary():
    x, t = rows(6, 5000, BF, 6)
    x[1] = math.nan
    t[1] = -1
    t[3], t[4] = 5000, -100
    x.requires_grad_()
    out = token_logprobs(x, t, top_k=3, ignore_index=-1)
    (dx,) = torch.autograd.grad([out.logprob.nan_to_num(0), out.entropy, out.top_logprob], x, [torch.ones(6, device="cuda")] * 2
                                + [torch.ones(6, 3, device="cuda")])
    assert out.logprob[1] == 0 and out.entropy[1] == 0 and out.top_index[1].tolist() == [-1] * 3 and not dx[1].any()
    assert out.logprob[3:5].isnan().all() and out.entropy[3:5].isfinite().all()
    assert not dx[[0, 2, 5]].isnan().any()


def test_parts_of_the_gradient():
    """Gradients that are absent or zero: the others alone; rows with none are not read."""
    x, t = rows(5, 3001, FP, 7)
    x.requires_grad_()
    for which in range(3):
        out = token_logprobs(x, t, top_k=4)
        gl, gh, gt = torch.zeros(5, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros(5, 4, device="cuda")
        given = (gl, gh, gt)[which]
        given += torch.randn_like(given)
        (dx,) = torch.autograd.grad(out[which], x, given)
        want, size = gradient(x.detach(), t, 1.0, 4, gl, gh, gt)
        tol = value_tolerance(x.detach(), 1.0)
        assert ((dx.double() - want).abs() <= want.abs() * HALF_STEP[FP] + size * 8 * tol * 10 + 2.0 ** -126).all()
    y = x.detach().clone()
    y[2] = math.nan
    y.requires_grad_()
    g = torch.ones(5, device="cuda")
    g[2] = 0
    (dy,) = torch.autograd.grad(token_logprobs(y, t).logprob, y, g)
    assert not dy[2].any() and dy[[0, 1, 3, 4]].any(1).all()
    # a gradient that can be differentiated again is the same gradient
    for which in range(3):
        g = torch.randn_like(token_logprobs(x, t, top_k=4)[which])
        (a,) = torch.autograd.grad(token_logprobs(x, t, top_k=4)[which], x, g)
        (b,) = torch.autograd.grad(token_logprobs(x, t, top_k=4)[which], x, g, create_graph=True)
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)
        assert torch.autograd.grad(b.square().sum(), x)[0].isfinite().all()


def test_batched_gradients():
    x, t = rows(3, 500, FP, 8)
    x.requires_grad_()
    out = token_logprobs(x, t, top_k=2)
    gs = torch.randn(4, 3, device="cuda")
    (got,) = torch.autograd.grad(out.logprob, x, gs, is_grads_batched=True, retain_graph=True)
    each = torch.stack([torch.autograd.grad(out.logprob, x, g, retain_graph=True)[0] for g in gs])
    torch.testing.assert_close(got, each, rtol=1e-5, atol=1e-6)


def test_captured_with_backward_on_another_stream():
    x, t = rows(30, 20000, BF, 9)
    x = x.clone().requires_grad_()
    eager = token_logprobs(x, t, temperature=0.8, top_k=5)
    g = [torch.randn(30, device="cuda"), torch.randn(30, device="cuda"), torch.randn(30, 5, device="cuda")]
    (want,) = torch.autograd.grad(list(eager[:3]), x, g)
    del eager
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = token_logprobs(x, t, temperature=0.8, top_k=5)
        torch.autograd.grad(list(out[:3]), x, g)
        del out
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = token_logprobs(x, t, temperature=0.8, top_k=5)
            (dx,) = torch.autograd.grad(list(out[:3]), x, g)
    torch.cuda.current_stream().wait_stream(side)
    dx.zero_()
    for _ in range(2):
        graph.replay()
    assert torch.equal(dx, want)
    ops.check_status()


def test_results_do_not_change_from_call_to_call():
    x, t = rows(64, 128256, BF, 10)
    x[::2, ::5] = 4.0
    first = token_logprobs(x, t, top_k=20)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, token_logprobs(x, t, top_k=20)))


def test_rows_far_apart():
    """Row offsets that pass 32 bits (a cache of logits, of which every millionth row is scored)."""
    ld, V = 1_100_000_008, 5001
    base = torch.empty(2 * ld + V + 3, dtype=BF, device="cuda")
    x = base[3:].as_strided((3, V), (ld, 1))
    g = torch.Generator(device="cuda").manual_seed(11)
    x.copy_(torch.randn(3, V, generator=g, device="cuda") * 3)
    check(x, torch.tensor([5, 5000, 0], device="cuda"), 1.0, 4)


@pytest.mark.parametrize("V,period,held,dtype", [(40000, 2048, 992, BF), (8000, 1024, 496, BF), (40000, 1024, 496, FP), (120000, 2048, 992, HF)])
def test_large_logits_that_few_threads_hold(V, period, held, dtype):
    """Rows whose large logits all fall to less than half of the threads, so that neither all above the bound on the
    alternatives nor all equal to it fit the candidates; with many equal ones, and with none."""
    g = torch.Generator(device="cuda").manual_seed(12)
    where = torch.arange(V, device="cuda") % period < held
    x = torch.zeros(3, V, device="cuda")
    x[0, where] = 1 + torch.rand(int(where.sum()), generator=g, device="cuda")
    x[1, where] = 2.0
    x[2] = torch.randn(V, generator=g, device="cuda") - 20
    x[2, where] += 30
    for k in (31, 32):
        check(x.to(dtype), torch.tensor([3, V - 1, 7], device="cuda"), 1.0, k)


@pytest.mark.parametrize("B,S,V,dtype", [(3, 5, 1000, BF), (2, 9, 1001, BF), (4, 2, 33, FP), (2, 700, 4096, HF), (1, 6, 500, BF)])
def test_batches_of_rows_where_they_lie(B, S, V, dtype):
    """All positions but the last of every sequence, and every second one: the same numbers as from a copy, without one. Rows that
    start elsewhere within 16 bytes than the copy's (an odd vocabulary) are added in another order: twice the sums' error."""
    g = torch.Generator(device="cuda").manual_seed(13)
    logits = (torch.randn(B, S + 1, V, generator=g, device="cuda") * 3).to(dtype)
    t = torch.randint(0, V, (B, S), generator=g, device="cuda")
    t[0, 0] = -100
    for view in (logits[:, :-1], logits[:, 1:], logits.repeat(1, 2, 1)[:, ::2][:, :S], logits.transpose(0, 1)[:S].transpose(0, 1)):
        x, y = view.detach().requires_grad_(), view.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        a, b = token_logprobs(x, t, top_k=3), token_logprobs(y, t, top_k=3)
        w = [torch.randn(o.shape, generator=g, device="cuda") for o in a[:3]]
        (dx,), (dy,) = torch.autograd.grad(a[:3], x, w), torch.autograd.grad(b[:3], y, w)
        assert dx.shape == view.shape and torch.equal(a.top_index, b.top_index)
        if V * x.element_size() % 16 == 0:
            assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(dx, dy)
            continue
        tol = 2 * value_tolerance(y.detach().view(-1, V), 1.0) * (1 + math.log(V))
        for p, q in zip(a[:3], b[:3]):
            torch.testing.assert_close(p, q, rtol=0, atol=tol)
        want, size = gradient(y.detach().view(-1, V), t.view(-1), 1.0, 3, w[0].view(-1), w[1].view(-1), w[2].view(-1, 3))
        for d in (dx, dy):
            off = (d.double().reshape(-1, V) - want).abs()
            assert (off <= want.abs() * HALF_STEP[dtype] + size * 8 * tol + SMALLEST[dtype]).all()
    before = torch.cuda.max_memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    now = torch.cuda.memory_allocated()
    with torch.no_grad():
        token_logprobs(logits[:, :-1], t)
    assert torch.cuda.max_memory_allocated() - now < logits[:, :-1].numel() * logits.element_size() // 2 + 65536, before
