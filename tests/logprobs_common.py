"""The definition of token log probabilities in 64 bits, and how far fp32 arithmetic may be from it."""
import math

import torch


def definition(x, target, temperature=1.0, k=0, ignore_index=-100):
    """(log probabilities [T, V], values dict) in 64 bits, from the formulas."""
    z = x.double() / temperature
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    s = e.sum(1, keepdim=True)
    lp = z - m - s.log()
    p = e / s
    H = -torch.where(p == 0, 0.0, p * torch.where(p == 0, 0.0, lp)).sum(1)
    live = target != ignore_index
    inside = live & (target >= 0) & (target < x.shape[1])
    at = torch.where(inside, target, 0)[:, None]
    # every NaN as one NaN: sorts by bit patterns take a negative one for the lowest value
    top = torch.sort(x.masked_fill(x.isnan(), math.nan), dim=1, descending=True, stable=True).indices[:, :k]
    out = {"logprob": torch.where(inside, lp.gather(1, at)[:, 0], torch.where(live, math.nan, 0.0)),
           "entropy": torch.where(live, H, 0.0), "top_logprob": torch.where(live[:, None], lp.gather(1, top), 0.0),
           "top_index": torch.where(live[:, None], top, -1)}
    return lp, out


def gradient(x, target, temperature, k, g, h, gt, ignore_index=-100):
    """(d logits, bound's p-weighted magnitude) of sum(g logprob + h entropy) + sum(gt top_logprob), in 64 bits."""
    lp, out = definition(x, target, temperature, k, ignore_index)
    live = target != ignore_index
    p, H = lp.exp(), out["entropy"][:, None]
    g, h, gt = g.double() * live, h.double() * live, gt.double() * live[:, None]
    flat = torch.where(p == 0, 0.0, lp)
    G = g + gt.sum(1)
    dz = -p * (G[:, None] + h[:, None] * (flat + H))
    dz.scatter_add_(1, torch.where(live, target, 0)[:, None], g[:, None])
    if k:
        dz.scatter_add_(1, torch.where(live[:, None], out["top_index"], 0), gt)
    size = p * (g.abs() + gt.abs().sum(1))[:, None] + p * h.abs()[:, None] * (flat.abs() + H + 1)
    dead = ~live[:, None]                   # ignored rows are not read, whatever they hold
    return dz.masked_fill(dead, 0.0) / temperature, size.masked_fill(dead, 0.0) / temperature


def value_tolerance(x, temperature):
    """Absolute error of a log probability. z = x / temperature carries two roundings, |z| 2^-23, and z - m one more; the sum
    of V exponentials adds V / 256 terms in a row at most (2^-24 each), then a tree of 16 and an exponential and a logarithm
    good to a few 2^-23 of their values. Entropies average such errors with weights that sum to 1 and up to ln V."""
    z = x.float()[x.isfinite() & (x.float().abs() < 1e30)].abs()
    top = float(z.max()) / temperature if z.numel() else 0.0
    V = x.shape[1]
    return (2 * top + 16 + math.log(V)) * 2.0 ** -22 + (V / 256 + 16) * 2.0 ** -24


# Relative error of a gradient besides what `gradient`'s second result scales. At a position that is the target and an
# alternative the kernel computes fl(fl(a) fl(1 / temperature) + ...) with a = fl(g + g_i): four fp32 roundings of 2^-24 each
# (sum, reciprocal, product, last sum), 2^-22 together; 16-bit gradients are rounded once more, by half a step.
FP32_STEPS = 2.0 ** -22
HALF_STEP = {torch.bfloat16: 2.0 ** -8 + FP32_STEPS, torch.float16: 2.0 ** -11 + FP32_STEPS, torch.float32: FP32_STEPS}
SMALLEST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}
