"""Rows of logits that lie far from zero, or far apart, once they are divided by the temperature, and how far fp32 arithmetic that
takes differences from the row's maximum may be from the definition. Nothing here grows with a common offset of the logits.

With u = 2^-24 (half a step of fp32), z = x / temperature, D_j = z_j - max z, p the distribution and E its mean:

* A difference (x_j - max x) / temperature carries three roundings (the subtraction, the reciprocal, the product): 3 u |D_j|.
* An exponential of it: its argument has four such roundings, the function is good to 2^-22 = 4 u, or as ``__expf`` to
  2 + 1.173 |D| units of 2 u each: less than (4 |D_j| + 8) u of its value.
* A thread adds n = V / 128 terms at most one after the other, as often rescales its sum (5 u, at most once in four terms of the
  same thread), and some sixteen such steps join the threads: (2 n + 70) u. So the sum s is good to
  sum_u = (4 E|D| + 2 n + 80) u, its logarithm to that and 4 (1 + ln V) u.
* log p_t = D_t - log s: ``log_tolerance``. H = log s + E|D|: the mean's terms |D_j| p_j carry the errors of |D_j| and of p_j
  as above, its quotient by s those of s: ``entropy_tolerance``.
* A derivative is p_j (G + h (log p_j + H)) / temperature and what a chosen position gets besides: relative errors of p_j as
  above, absolute ones of log p_j and H, (k + 6) roundings of the sums and products of the given gradients, and one to the
  logits' type."""
import math

import torch

from flex_shard_b200.ops.logprobs import token_logprobs
from tests.logprobs_common import definition, gradient

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALLEST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def check(x, t, temperature=1.0, k=0, grads=True):
    """Values, alternatives and gradients of finite rows [T, V]."""
    T, V = x.shape
    x = x.detach().requires_grad_(grads)
    out = token_logprobs(x, t, temperature=temperature, top_k=k)
    before = x.detach()
    lp, ref = definition(before, t, temperature, k)
    z = before.double() / temperature
    D = (z - z.amax(1, keepdim=True)).abs()
    p = lp.exp()
    mean = lambda v: torch.where(p == 0, 0.0, p * v).sum(1)  # noqa: E731
    ED, ED2 = mean(D), mean(D * D)
    n = V / 128 + 1
    log_u = (4 * ED + 2 * n + 84 + 4 * math.log(V)) * U
    ent_u = ((2 * n + 90) * (1 + 2 * ED) + 4 * ED2 + 8 * ED + 8 * math.log(V)) * U
    log_tolerance = lambda d: log_u.view(-1, *[1] * (d.dim() - 1)) + 4 * d * U  # noqa: E731
    assert torch.equal(out.top_index, ref["top_index"])
    pairs = [("logprob", ref["logprob"], log_tolerance(D.gather(1, t[:, None])[:, 0])), ("entropy", ref["entropy"], ent_u),
             ("top_logprob", ref["top_logprob"], log_tolerance(D.gather(1, ref["top_index"])) if k else torch.zeros(T, 0, device=x.device))]
    for name, want, tol in pairs:
        got = getattr(out, name).double()
        low = (want < -3.4e38) & (got == -math.inf)             # below the range of fp32
        off = torch.where(low, 0.0, got - want).abs()
        assert (off <= tol).all(), f"{name}: {float((off - tol).max())} beyond at temperature {temperature}"
    # what no rounding may take away
    assert (out.logprob <= 0).all() and (out.top_logprob <= 0).all() and (out.entropy >= 0).all()
    if not grads:
        return out
    g = torch.Generator().manual_seed(1)
    gl, gh, gt = (torch.randn(s, generator=g).to(x.device) for s in ((T,), (T,), (T, k)))
    (dx,) = torch.autograd.grad([out.logprob, out.entropy, out.top_logprob], x, [gl, gh, gt])
    want, _ = gradient(before, t, temperature, k, gl, gh, gt)
    G, h = (gl.abs() + gt.abs().sum(1)).double()[:, None], gh.abs().double()[:, None]
    l, H = torch.where(p == 0, 0.0, lp.abs()), ref["entropy"][:, None]
    rel = torch.where(p == 0, 0.0, 4 * D * U) + log_u[:, None] + (k + 8) * U
    bound = p * (G + h * (l + H)) * rel + p * h * (log_u + ent_u)[:, None] + torch.where(p == 0, 0.0, p * h * 4 * D * U)
    chosen = torch.zeros_like(bound).scatter_(1, t[:, None], 1.0)
    if k:
        chosen.scatter_(1, ref["top_index"], 1.0)
    bound = (bound + chosen * G * (k + 6) * U) / temperature
    lost = 2.0 ** -126 * (G + h * (88 + math.log(V))) / temperature   # probabilities below 2^-126 count as 0
    off = (dx.double() - want).abs()
    assert (off <= bound + want.abs() * HALF[x.dtype] + SMALLEST[x.dtype] + lost).all(), f"gradient at temperature {temperature}"
    return out


def randn(T, V, dtype, device, seed=0, scale=4.0, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, V, generator=g, dtype=torch.float64) * scale + offset).to(dtype)
    t = torch.randint(0, V, (T,), generator=g)
    t[0] = int(x[0].argmax())
    return x.to(device), t.to(device)


def low_temperatures(V, T, dtype, temperature, device):
    x, t = randn(T, V, dtype, device)
    check(x, t, temperature, min(V, 5), grads=dtype is not HF or temperature >= 0.01)     # fp16 holds no larger gradients


def common_offsets(V, dtype, offset, device):
    """Rows around one value: all digits that the type leaves of their differences count."""
    x, t = randn(4, V, dtype, device, 1, 3.0, offset)
    for temperature in (1.0, 0.7):
        check(x, t, temperature, min(V, 5))


def one_token(dtype, value, device):
    """A vocabulary of one token: a probability of exactly 1."""
    x, t = torch.full((3, 1), value, device=device).to(dtype), torch.zeros(3, dtype=torch.int64, device=device)
    for temperature in (1.0, 0.3, 1e-6, 1e6):
        out = check(x, t, temperature, 1)
        assert not out.logprob.any() and not out.entropy.any() and not out.top_logprob.any()


def equal_rows(V, dtype, value, device):
    x, t = torch.full((2, V), value, device=device).to(dtype), torch.tensor([0, V - 1], device=device)
    for temperature in (1.0, 0.01):
        check(x, t, temperature, min(V, 5))


def finite_masks(V, dtype, mask, device):
    """Masked by a finite number: half of the tokens, runs of them, all that some threads read, all but one, and single ones."""
    x, t = randn(6, V, dtype, device, 2)
    at = torch.arange(V, device=device)
    for row, where in enumerate((at % 2 == 0, (at > V // 3) & (at < V - 3), at % 2048 < 1500, at != V // 2, at == 7 % V)):
        x[row, where] = mask
        t[row] = int(x[row].argmax())
    t[5] = V - 1
    for temperature in (1.0, 0.05):
        check(x, t, temperature, min(V, 5), grads=dtype is not HF or temperature >= 0.01)
