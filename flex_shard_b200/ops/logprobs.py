"""Log probabilities of given tokens with the entropy of their distribution and its top alternatives, and their gradient
(``csrc/logprobs.cu``). The counterpart of ``cross_entropy`` where a value per token is wanted: policy gradients,
distillation on a teacher's alternatives, scoring.

CPU tensors take a PyTorch restatement of the same arithmetic, and so do ``torch.func`` transforms, forward-mode derivatives,
batched gradients and gradients that are differentiated again.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import count_launch

MAX_TOP_K = 32
_KINDS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_declared = False


class TokenLogprobs(NamedTuple):
    """``logprob`` and ``entropy`` (nats) have the target's shape, ``top_logprob`` and ``top_index`` one more axis of length
    ``top_k``, best first. fp32, and int64 for the indices."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor
    top_index: torch.Tensor


def _ensure():
    global _declared
    if not _declared:
        c = ctypes
        vp, i32, i64, f32 = c.c_void_p, c.c_int, c.c_longlong, c.c_float
        _lib.declare("fsb_token_logprobs", [vp, i32, vp, i64, i32, i64, i64, i64, f32, i32, i64, vp, vp, vp, vp, vp, vp])
        _lib.declare("fsb_token_logprobs_bwd", [vp, i32, vp, i64, i32, i64, i64, i64, f32, i32, i64, vp, vp, vp, vp, vp, vp, vp, i64, vp])
        _declared = True


def _top_indices(x: torch.Tensor, k: int) -> torch.Tensor:
    """The k largest of every row, best first; the lower index first among equals (a NaN counts as the largest)."""
    x = x.masked_fill(x.isnan(), float("nan"))      # a device's sort may take a negative NaN for the lowest value
    return torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]


def _restatement(x, target, temperature, k, ignore_index):
    """The operator in differentiable PyTorch operations."""
    V = x.shape[-1]
    x = x.reshape(-1, V)
    live = target != ignore_index
    valid = live & (target >= 0) & (target < V)
    xf = torch.where(live[:, None], x, 0).float()       # ignored rows take no part, whatever they hold
    lp = torch.log_softmax((xf - xf.detach().amax(-1, keepdim=True)) / temperature, -1)
    at = torch.where(valid, target, 0)
    # a target outside the vocabulary makes its row's value and gradient NaN
    logprob = torch.where(live, lp.gather(1, at[:, None]).squeeze(1) * torch.where(live & ~valid, torch.nan, 1.0), 0.0)
    # 0 log 0 counts as 0; a NaN (no distribution) stays one
    p = lp.exp()
    plogp = torch.where(p == 0, 0.0, p * torch.where(p == 0, 0.0, lp))
    entropy = torch.where(live, -plogp.sum(-1), 0.0)
    top = _top_indices(x.detach(), k)
    top_logprob = torch.where(live[:, None], lp.gather(1, top), 0.0)
    return logprob, entropy, top_logprob, torch.where(live[:, None], top, -1)


def _restated_gradient(x, target, top, stats, entropy, temperature, ignore_index, glp, gh, gtop):
    """The gradient's formula in PyTorch operations (gradients may be batched)."""
    shape, V = x.shape, x.shape[-1]
    x = x.reshape(-1, V)
    live = target != ignore_index
    valid = live & (target >= 0) & (target < V)
    lp = (x.float() - stats[:, :1]) / temperature - stats[:, 1:]
    p = lp.exp()
    cols = torch.arange(V, device=x.device)
    dz = torch.zeros((), device=x.device)
    wanted = torch.zeros((), dtype=torch.bool, device=x.device)
    if glp is not None:
        nan = torch.where(live & ~valid, torch.nan, 0.0)[:, None]
        dz = dz + glp[:, None] * ((cols == torch.where(valid, target, 0)[:, None]).float() - p + nan)
        wanted = wanted | (glp != 0)
    if gh is not None:
        dz = dz - gh[:, None] * torch.where(p == 0, 0.0, p * (torch.where(p == 0, 0.0, lp) + entropy[:, None]))
        wanted = wanted | (gh != 0)
    if gtop is not None:
        for i in range(top.shape[1]):
            dz = dz + gtop[:, i, None] * ((cols == top[:, i, None]).float() - p)
            wanted = wanted | (gtop[:, i] != 0)
    return (torch.where((live & wanted)[:, None], dz, 0.0) / temperature).to(x.dtype).reshape(shape)


def _rows(x):
    """How the kernels find the rows of ``[T, V]`` or ``[batches, rows, V]`` logits."""
    return (0, 0, x.stride(0)) if x.dim() == 2 else (x.shape[1], x.stride(0), x.stride(1))


def _forward(x, target, temperature, k, ignore_index, stats):
    """``x`` is ``[T, V]`` or ``[batches, rows, V]`` with ``T`` rows in all. ``stats`` [T, 2] takes the numbers of a row that the gradient starts from, the largest logit and the logarithm of the
    sum relative to it (``None``: not wanted)."""
    T, V = target.shape[0], x.shape[-1]
    if not x.is_cuda:
        if stats is not None:
            xf = x.reshape(-1, V).float()
            m = xf.amax(-1, keepdim=True)
            stats.copy_(torch.cat([m, ((xf - m) / temperature).exp().sum(-1, keepdim=True).log()], -1))
        return _restatement(x, target, temperature, k, ignore_index)
    _ensure()
    dev = x.device
    logprob = torch.empty(T, dtype=torch.float32, device=dev)
    entropy = torch.empty(T, dtype=torch.float32, device=dev)
    top_lp = torch.empty(T, k, dtype=torch.float32, device=dev)
    top = torch.empty(T, k, dtype=torch.int64, device=dev)
    with _lib.device_of(x):
        rc = _lib.load().fsb_token_logprobs(x.data_ptr(), _KINDS[x.dtype], target.data_ptr(), T, V, *_rows(x), 1.0 / temperature,
                                            k, ignore_index, logprob.data_ptr(), entropy.data_ptr(),
                                            None if stats is None else stats.data_ptr(), top_lp.data_ptr(), top.data_ptr(),
                                            _lib.stream_ptr(dev))
    _lib.check(rc, "fsb_token_logprobs")
    count_launch(int(T > 0))
    return logprob, entropy, top_lp, top


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, target, temperature, k, ignore_index):
        stats = torch.empty(target.shape[0], 2, dtype=torch.float32, device=x.device)
        logprob, entropy, top_lp, top = _forward(x, target, temperature, k, ignore_index, stats)
        ctx.save_for_backward(x, target, top, stats, entropy)
        ctx.cfg = (temperature, ignore_index)
        ctx.mark_non_differentiable(top)
        ctx.set_materialize_grads(False)
        return logprob, entropy, top_lp, top

    @staticmethod
    def backward(ctx, glp, gh, gtop, _):
        x, target, top, stats, entropy = ctx.saved_tensors
        temperature, ignore_index = ctx.cfg
        T, V = target.shape[0], x.shape[-1]
        k = top.shape[1]
        if k == 0:
            gtop = None
        given = [g for g in (glp, gh, gtop) if g is not None]
        if not given:
            return None, None, None, None, None
        if torch.is_grad_enabled():     # a gradient that may be differentiated again: PyTorch's own derivatives
            outs = _restatement(x, target, temperature, k, ignore_index)
            (dx,) = torch.autograd.grad([o for o, g in zip(outs, (glp, gh, gtop)) if g is not None], x, given, create_graph=True)
            return dx, None, None, None, None
        if not x.is_cuda or not _lib.plain(*given):
            return _restated_gradient(x, target, top, stats, entropy, temperature, ignore_index, glp, gh, gtop), None, None, None, None
        glp, gh, gtop = (None if g is None else g.float().contiguous() for g in (glp, gh, gtop))
        # rows of the gradient start as far into 16 bytes as the logits' rows do, so that both move in whole vectors
        lanes = 16 // x.element_size()
        ld = V + (x.stride(-2) - V) % lanes if T > 1 else V
        dx = torch.empty(*x.shape[:-1], ld, dtype=x.dtype, device=x.device)[..., :V]
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        with _lib.device_of(x):
            rc = _lib.load().fsb_token_logprobs_bwd(x.data_ptr(), _KINDS[x.dtype], target.data_ptr(), T, V, *_rows(x),
                                                    1.0 / temperature, k, ignore_index, top.data_ptr(), stats.data_ptr(),
                                                    entropy.data_ptr(), ptr(glp), ptr(gh), ptr(gtop), dx.data_ptr(), ld,
                                                    _lib.stream_ptr(x.device))
        _lib.check(rc, "fsb_token_logprobs_bwd")
        count_launch(int(T > 0))
        return dx, None, None, None, None


def token_logprobs(logits: torch.Tensor, target: torch.Tensor, *, temperature: float = 1.0, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """``log softmax(logits / temperature)`` at ``target``, the distribution's entropy and its ``top_k`` likeliest tokens.

    ``logits [..., V]`` bf16, fp16 or fp32 (strided rows, and batches of rows such as ``logits[:, :-1]``, are read where they
    lie), ``target [...]`` integer; ``top_k`` up to 32 and V. All
    arithmetic in fp32; the logits are read once and left as they are. Differentiable with respect to ``logits`` through
    ``logprob``, ``entropy`` and ``top_logprob`` (the choice of alternatives counts as constant); the backward pass reads the
    logits again, so they must not be overwritten before it (as ``cross_entropy`` does).

    * Errors grow with a logit's distance from the row's largest over the temperature, not with what the row's logits share; log
      probabilities are at most 0, entropies at least 0, and both exactly 0 where one token is left. On the GPU a row whose
      largest logit over the temperature is beyond 4.6e7 in magnitude is read four times instead of once.
    * Alternatives are ordered by logit, the lower index first among equals; a NaN counts as the largest.
    * Rows whose target is ``ignore_index`` are not read: 0 for all values, -1 for the indices, no gradient.
    * Any other target outside the vocabulary gives a NaN log probability (entropy and alternatives are unaffected).
    * Logits of minus infinity have probability 0 and add nothing. A row without a distribution (all minus infinity, a plus
      infinity, a NaN) gives NaN, as ``log_softmax`` does.
    * A row whose gradients are all exactly 0 gets a gradient of 0 without being read."""
    if logits.dim() < 1 or logits.shape[:-1] != target.shape:
        raise ValueError(f"target {tuple(target.shape)} does not match logits {tuple(logits.shape)} ([..., V])")
    if logits.dtype not in _KINDS:
        raise ValueError(f"logits must be bf16, fp16 or fp32, got {logits.dtype}")
    if target.is_floating_point() or target.is_complex() or target.dtype == torch.bool:
        raise ValueError(f"target must hold integers, got {target.dtype}")
    if target.device != logits.device:
        raise ValueError(f"target is on {target.device}, logits on {logits.device}")
    V = logits.shape[-1]
    if V < 1:
        raise ValueError("the vocabulary is empty")
    if not 0 <= top_k <= min(MAX_TOP_K, V):
        raise ValueError(f"top_k must be between 0 and {min(MAX_TOP_K, V)} (at most {MAX_TOP_K}, and the vocabulary), got {top_k}")
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:        # its reciprocal is an fp32 number
        raise ValueError(f"temperature must be positive and finite (1e-30 to 1e30), got {temperature}")
    lead = target.shape
    x, t = logits, target
    if len(lead) != 1:
        t = t.reshape(-1)
        # batches of rows (all positions but a sequence's last, for instance) are taken where they lie
        if not (len(lead) == 2 and x.is_cuda and x.stride(2) == 1 and x.stride(0) != lead[1] * x.stride(1) and t.numel()):
            x = x.reshape(-1, V)
    if t.dtype != torch.int64:
        t = t.long()
    if _lib.plain(logits, target) and forward_ad._current_level < 0:
        if V > 1 and x.stride(-1) != 1:
            x = x.contiguous()
        if not t.is_contiguous():
            t = t.contiguous()
        if logits.requires_grad and torch.is_grad_enabled():
            out = _TokenLogprobs.apply(x, t, temperature, top_k, ignore_index)
        else:
            out = _forward(x, t, temperature, top_k, ignore_index, None)
    else:
        out = _restatement(x, t, temperature, top_k, ignore_index)
    if len(lead) != 1:
        out = (out[0].view(lead), out[1].view(lead), out[2].view(*lead, top_k), out[3].view(*lead, top_k))
    return TokenLogprobs(*out)
