"""Token log probabilities on CPU tensors: the definition, its gradient against differences, and the refusals."""
import math

import pytest
import torch

from flex_shard_b200.ops.logprobs import TokenLogprobs, token_logprobs
from tests.logprobs_common import HALF_STEP, definition, gradient, value_tolerance


def rows(T, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, V, generator=g) * 3).to(dtype)
    return x, torch.randint(0, V, (T,), generator=g)


@pytest.mark.parametrize("T,V,k,temperature,dtype", [(1, 1, 1, 1.0, torch.float32), (5, 33, 4, 0.7, torch.bfloat16),
                                                     (9, 1000, 32, 1.5, torch.float16), (3, 77, 0, 1.0, torch.float32)])
def test_values_and_gradient(T, V, k, temperature, dtype):
    x, t = rows(T, V, dtype)
    if T > 2:
        t[2] = -100
        x[1, : V // 2] = -math.inf
        t[1] = V - 1
    x.requires_grad_()
    out = token_logprobs(x, t, temperature=temperature, top_k=k)
    _, ref = definition(x.detach(), t, temperature, k)
    tol = value_tolerance(x.detach(), temperature)
    for name in ("logprob", "entropy", "top_logprob"):
        torch.testing.assert_close(getattr(out, name).double(), ref[name].double(), rtol=0, atol=tol * (1 + math.log(V)))
    assert torch.equal(out.top_index, ref["top_index"])
    g = torch.Generator().manual_seed(1)
    gl, gh, gt = (torch.randn(n, generator=g) for n in ((T,), (T,), (T, k)))
    (dx,) = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, [gl, gh, gt])
    want, size = gradient(x.detach(), t, temperature, k, gl, gh, gt)
    assert ((dx.double() - want).abs() <= want.abs() * HALF_STEP[dtype] + size * 8 * tol * (1 + math.log(V)) + 2.0 ** -24).all()


def test_the_formula_of_the_gradient_against_differences():
    """Central differences in 64 bits: truncation h^2 |f'''| / 6 (f''' below 40 for values of this size) and cancellation
    2^-52 |f| / h with |f| < 100 leave 1e-6 at h = 1e-4."""
    x, t = rows(4, 17, torch.float64)
    t[3] = -100
    g = torch.Generator().manual_seed(2)
    gl, gh, gt = (torch.randn(n, generator=g, dtype=torch.float64) for n in ((4,), (4,), (4, 5)))

    def value(x):
        _, o = definition(x, t, 0.8, 5)
        return float((gl * o["logprob"]).sum() + (gh * o["entropy"]).sum() + (gt * o["top_logprob"]).sum())

    want, _ = gradient(x, t, 0.8, 5, gl, gh, gt)
    for i in range(4):
        for j in range(17):
            a, b = x.clone(), x.clone()
            a[i, j] += 1e-4
            b[i, j] -= 1e-4
            assert abs((value(a) - value(b)) / 2e-4 - float(want[i, j])) < 1e-6


def test_rows_without_a_distribution_and_odd_targets():
    x, t = rows(6, 20, torch.float32)
    x[0] = -math.inf
    x[1, 3] = math.inf
    x[2, 4] = math.nan
    t[3], t[4] = 20, -7
    t[5] = -100
    out = token_logprobs(x, t, top_k=2)
    assert isinstance(out, TokenLogprobs)
    assert out.logprob[:5].isnan().all() and out.entropy[:3].isnan().all() and out.entropy[3:5].isfinite().all()
    assert out.top_index[0].tolist() == [0, 1] and out.top_index[1, 0] == 3 and out.top_index[2, 0] == 4
    assert out.logprob[5] == 0 and out.entropy[5] == 0 and out.top_index[5].tolist() == [-1, -1]


def test_gradients_of_odd_rows():
    """A row whose gradients are all 0 has none, whatever its logits; a target outside the vocabulary makes its row NaN."""
    x, t = rows(4, 20, torch.float32)
    x[0], t[1], t[3] = math.nan, 25, -100
    x.requires_grad_()
    out = token_logprobs(x, t, top_k=2)
    (dx,) = torch.autograd.grad(out.logprob, x, torch.tensor([0.0, 1.0, 1.0, 1.0]))
    assert not dx[0].any() and dx[1].isnan().all() and dx[2].isfinite().all() and dx[2].any() and not dx[3].any()


def test_second_derivatives():
    """Of the values' sum along a direction, against automatic differentiation of the definition in 64 bits: a few hundred fp32
    operations on numbers of order 1."""
    x, t = rows(4, 13, torch.float32)
    t[1] = -100
    x[1] = math.nan
    v = torch.randn(4, 13)
    w = torch.randn(3)

    def second(z, f):
        z = z.requires_grad_()
        o = f(z)
        total = w[0] * o[0].sum() + w[1] * (o[1] * o[1]).sum() + w[2] * o[2].sum()
        (d,) = torch.autograd.grad(total, z, create_graph=True)
        return torch.autograd.grad((d * v).sum(), z)[0]

    got = second(x.clone(), lambda z: token_logprobs(z, t, temperature=0.9, top_k=3))

    def plain(z):
        keep = [0, 2, 3]
        lp = torch.log_softmax(z[keep] / 0.9, -1)
        return (lp.gather(1, t[keep][:, None]), -(lp.exp() * lp).sum(-1), lp.topk(3).values)

    want = second(x.double(), plain)
    assert not got[1].any()
    torch.testing.assert_close(got[[0, 2, 3]].double(), want[[0, 2, 3]], rtol=1e-4, atol=1e-4)


def test_transforms_and_forward_derivatives_take_the_restatement():
    x, t = rows(3, 11, torch.float32)
    f = lambda z: token_logprobs(z, t, top_k=2).logprob.sum()  # noqa: E731
    want = gradient(x, t, 1.0, 2, torch.ones(3), torch.zeros(3), torch.zeros(3, 2))[0]
    torch.testing.assert_close(torch.func.grad(f)(x).double(), want, rtol=0, atol=1e-5)
    v = torch.randn(3, 11)
    torch.testing.assert_close(torch.func.jvp(f, (x,), (v,))[1].double(), (want * v).sum(), rtol=0, atol=1e-4)


def test_leading_axes_and_equal_logits():
    x = torch.zeros(2, 3, 40)
    x[..., 7] = -0.0
    out = token_logprobs(x, torch.ones(2, 3, dtype=torch.int32), top_k=9)
    assert out.logprob.shape == (2, 3) and out.top_index.shape == (2, 3, 9)
    assert (out.top_index == torch.arange(9)).all()
    torch.testing.assert_close(out.entropy, torch.full((2, 3), math.log(40)))


def test_refusals():
    x, t = rows(4, 20, torch.float32)
    for kw, text in ((dict(top_k=21), "top_k"), (dict(top_k=-1), "top_k"), (dict(temperature=0.0), "temperature"),
                     (dict(temperature=math.nan), "temperature"), (dict(temperature=math.inf), "temperature")):
        with pytest.raises(ValueError, match=text):
            token_logprobs(x, t, **kw)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(torch.zeros(4, 50), t, top_k=33)
    with pytest.raises(ValueError, match="does not match"):
        token_logprobs(x, t[:3])
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        token_logprobs(x.double(), t)
    with pytest.raises(ValueError, match="integers"):
        token_logprobs(x, t.float())
    with pytest.raises(ValueError, match="empty"):
        token_logprobs(x[:, :0], t)
