"""The 4-bit linear and token log-probability operators of this framework, as cases that can be timed and compared.

``own`` false: plain forms in elementary torch operations. ``own`` true: the framework's entry points
(``flex_shard_b200.ops.mxfp4``, ``flex_shard_b200.ops.logprobs``). A case is one call as a user's program makes it:

* ``quantise``: activations (32-element groups of a row) or a weight (32x32 tiles) to MXFP4, returned as the values the
  codes stand for;
* ``linear``: a frozen 4-bit weight applied to bf16 rows, from one token to a long batch;
* ``train``: the 4-bit linear with its weight quantised on the way, forward and both gradients;
* ``score``: log probabilities of given tokens, entropy and top alternatives;
* ``policy``: the same with the gradient of the logits.
"""
from __future__ import annotations

import math

import torch

own = False
GPU = torch.device("cuda")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------------------- the cases
def _quantise(name, rows, cols, weight):
    return dict(name=name, kind="quantise", rows=rows, cols=cols, weight=weight)


def _linear(name, T, N, K):
    return dict(name=name, kind="linear", T=T, N=N, K=K)


def _train(name, T, N, K):
    return dict(name=name, kind="train", T=T, N=N, K=K)


def _logprobs(name, kind, T, V, dtype="bf16", k=0, temperature=1.0, masked=0.0, ignored=0.0):
    return dict(name=name, kind=kind, T=T, V=V, dtype=dtype, k=k, temperature=temperature, masked=masked, ignored=ignored)


def listed():
    return [
        # the input of a down projection, an odd number of tokens
        _quantise("quantise_rows", 5765, 14336, False),
        # a gate / up weight whose rows end inside a tile
        _quantise("quantise_weight", 28660, 4096, True),
        # the next token of one sequence through a fused query / key / value projection
        _linear("linear_token", 1, 6144, 4096),
        # next tokens of a batch of sequences through the gate / up projection
        _linear("linear_batch", 48, 28672, 4096),
        # a short ragged prompt, output and input widths that no tile divides
        _linear("linear_ragged", 777, 5000, 2080),
        # a long prompt or an evaluation batch through the gate / up projection
        _linear("linear_long", 8192, 28672, 4096),
        # a training step of a small square projection
        _train("train_small", 500, 2048, 2048),
        # a training step of the down projection at the benchmark's sequence length
        _train("train_long", 8192, 4096, 14336),
        # next-token scores of a few sequences: one wave of rows, twenty alternatives each
        _logprobs("score_few", "score", 7, 128256, k=20, temperature=0.7),
        # a teacher scoring a whole batch: eight alternatives, a third of the vocabulary masked
        _logprobs("score_batch", "score", 8192, 128256, k=8, masked=0.33),
        # a policy-gradient step with an entropy bonus; prompt rows are ignored
        _logprobs("policy_batch", "policy", 4096, 102400, temperature=0.9, ignored=0.3),
        # distillation on the teacher's alternatives in fp32, an odd vocabulary
        _logprobs("policy_odd", "policy", 1500, 50021, dtype="fp32", k=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "linear", "linear", "train", "score", "policy"])
    if kind == "quantise":
        cols = 32 * _log(rng, 2, 512)
        rows = _log(rng, 1, min(32768, 28660 * 4096 // cols))
        case = _quantise("", rows, cols, rng.random() < 0.5)
    elif kind == "linear":
        T, K = _log(rng, 1, 8192), 32 * _log(rng, 2, 448)
        N = _log(rng, 16, min(32768, 8192 * 28672 * 4096 // (T * K)))
        case = _linear("", T, N, K)
    elif kind == "train":
        T, K = _log(rng, 1, 8192), 128 * _log(rng, 1, 112)
        if rng.random() < 0.5:
            T = -(-T // 128) * 128
        N = 128 * _log(rng, 1, min(112, 8192 * 4096 * 14336 // (T * K * 128)))
        case = _train("", T, N, K)
    else:
        V = _log(rng, 100, 160000)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = (8192 * 128256 if kind == "score" else 4096 * 102400) // (2 if dtype == "fp32" else 1)
        T = _log(rng, 1, min(8192, most // V))
        case = _logprobs("", kind, T, V, dtype, rng.choice([0, 1, 5, 8, 20, 32]), rng.choice([1.0, 1.0, 0.6, 1.3]),
                         rng.choice([0.0, 0.0, 0.5]), rng.choice([0.0, 0.2]))
    del case["name"]
    return case


# --------------------------------------------------------------------------- what a user's program has in hand
def _activations(g, rows, cols):
    """Rows of a residual stream at work: uneven token norms and a few outlying channels."""
    x = torch.randn(rows, cols, generator=g, device=GPU)
    x *= 0.5 + torch.rand(rows, 1, generator=g, device=GPU)
    x *= torch.where(torch.rand(cols, generator=g, device=GPU) < 0.01, 8.0, 1.0)
    return x.to(torch.bfloat16)


def _weight(g, rows, cols):
    return (torch.randn(rows, cols, generator=g, device=GPU) / math.sqrt(cols)).to(torch.bfloat16)


def _pack(codes):
    return codes[:, 0::2] | codes[:, 1::2] << 4


def _blocked(scales):
    """The tensor core's order of scale bytes: blocks of 128 rows x 4 groups, 512 bytes each."""
    rows, groups = scales.shape
    full = torch.full((-(-rows // 128) * 128, -(-groups // 4) * 4), 127, dtype=torch.uint8, device=scales.device)
    full[:rows, :groups] = scales
    return full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def prepare(case, seed):
    g = torch.Generator(device=GPU).manual_seed(seed)
    kind, state = case["kind"], {"case": case}
    if kind == "quantise":
        state["x"] = (_weight if case["weight"] else _activations)(g, case["rows"], case["cols"])
    elif kind == "linear":
        state["x"] = _activations(g, case["T"], case["K"])
        # the frozen weight as the program keeps it: packed codes and tile exponents, and the scales in the tensor core's order
        codes, exponents = _codes(_weight(g, case["N"], case["K"]), 32)
        state["codes"], state["exponents"] = _pack(codes), exponents
        state["scales"] = _blocked(exponents.repeat_interleave(32, 0)[:case["N"]])
    elif kind == "train":
        state["x"] = _activations(g, case["T"], case["K"]).requires_grad_()
        state["w"] = _weight(g, case["N"], case["K"]).requires_grad_()
        state["dy"] = (torch.randn(case["T"], case["N"], generator=g, device=GPU) * 1e-3).to(torch.bfloat16)
    else:
        T, V, k = case["T"], case["V"], case["k"]
        dtype = DTYPES[case["dtype"]]
        logits = torch.empty(T, V, dtype=dtype, device=GPU)
        step = max(1, (1 << 27) // V)
        for i in range(0, T, step):                      # rows of different sharpness
            part = torch.randn(min(step, T - i), V, generator=g, device=GPU)
            part *= 1.0 + 2.0 * torch.rand(part.shape[0], 1, generator=g, device=GPU)
            logits[i:i + step] = part
        target = torch.randint(0, V, (T,), generator=g, device=GPU)
        if case["masked"]:
            banned = torch.rand(V, generator=g, device=GPU) < case["masked"]
            banned[:64] = False
            logits[:, banned] = -math.inf
            target = torch.where(banned[target], target % 64, target)
        if case["ignored"]:
            target[torch.rand(T, generator=g, device=GPU) < case["ignored"]] = -100
        state["logits"], state["target"] = logits, target
        if kind == "policy":
            logits.requires_grad_()
            state["d_logprob"] = torch.randn(T, generator=g, device=GPU) / T
            state["d_entropy"] = torch.full((T,), -0.01 / T, device=GPU)
            state["d_top"] = torch.rand(T, k, generator=g, device=GPU) / -T
    return state


# --------------------------------------------------------------------------- plain forms
def _power(byte):
    """2^(byte - 127), exactly, for bytes 0 to 254."""
    byte = byte.to(torch.int32)
    return torch.where(byte == 0, torch.full_like(byte, 1 << 22), byte << 23).view(torch.float32)


def _groups(x, block):
    """Tiles of ``block`` x 32 elements, padded with zeros: [row blocks, block, column groups, 32]."""
    rows, cols = x.shape
    pad = torch.zeros(-(-rows // block) * block, cols, dtype=torch.float32, device=x.device)
    pad[:rows] = x
    return pad.view(-1, block, cols // 32, 32)


def _codes(x, block):
    """MXFP4 codes [rows, cols] (uint8, 4 bits used) and scale bytes [row blocks, column groups] of tiles of block x 32."""
    t = _groups(x.detach(), block)
    bits = t.abs().amax(dim=(1, 3)).view(torch.int32)
    e = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x400000).int()).clamp_min(0)
    v = t * _power(254 - e)[:, None, :, None]
    a = v.abs()
    # midpoints between the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6; a tie goes to the even code
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + (v < 0).to(torch.uint8) * 8
    return code.view(-1, x.shape[1])[:x.shape[0]].contiguous(), e.to(torch.uint8)


def _values(codes, scales, block):
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    rows = codes.shape[0]
    s = _power(scales).repeat_interleave(block, 0)[:rows].repeat_interleave(32, 1)
    return table[codes.int()] * s


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], -1).view(packed.shape[0], -1)


def _mx8(x, dim):
    """The values of MXFP8 (e4m3, groups of 32 along ``dim``, scale the smallest power of two with amax / s <= 448)."""
    t = x.detach().float()
    t = t.t().contiguous() if dim == 0 else t
    t = t.view(t.shape[0], -1, 32)
    bits = (t.abs().amax(-1) * (1.0 / 448.0)).view(torch.int32)
    e = bits >> 23
    e = torch.where((bits & 0x7FFFFF) != 0, e + 1, e) * (bits != 0)
    q = (t * _power(254 - e)[..., None]).to(torch.float8_e4m3fn).float() * _power(e)[..., None]
    q = q.view(q.shape[0], -1)
    return q.t() if dim == 0 else q


def _plain_quantise(x, weight):
    block = 32 if weight else 1
    codes, e = _codes(x, block)
    out = {"values": _values(codes, e, block).to(torch.bfloat16)}
    if weight:
        out["exponents"] = e
    return out


def _plain_train(x, w, dy):
    w4 = _values(*_codes(w, 32), 32)
    y = _values(*_codes(x, 1), 1) @ w4.t()
    dx = _mx8(dy, 1) @ w4
    if x.shape[0] % 128 == 0:
        dw = _mx8(dy, 0).t() @ _mx8(x, 0)
    else:
        dw = dy.float().t() @ x.detach().float()
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw.to(w.dtype)}


def _ordered_key(x):
    """Whole numbers that order like the floats of x, the lower index first among equals, all different."""
    bits = (x.float() + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return bits * (1 << 20) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))


def _plain_logprobs(case, logits, target, d=None):
    """Row blocks, so that the 32-bit temporaries stay small."""
    T, V, k, tau = case["T"], case["V"], case["k"], case["temperature"]
    parts = []
    step = max(1, (1 << 26) // V)
    for i in range(0, T, step):
        x, t = logits.detach()[i:i + step], target[i:i + step]
        live = t != -100
        top = V - 1 - _ordered_key(x).topk(k, dim=1).values % (1 << 20) if k else t[:, None][:, :0]
        z = x.float() / tau
        zt, ztop = z.gather(1, t.clamp_min(0)[:, None]).squeeze(1), z.gather(1, top)
        m = z.amax(1, keepdim=True)
        z -= m
        p = z.exp()
        s = p.sum(1, keepdim=True)
        p /= s
        z = torch.where(p > 0, z, torch.zeros_like(z))
        log_s = s.log()
        entropy = (log_s - (p * z).sum(1, keepdim=True)).squeeze(1)
        lse = m + log_s
        out = {"logprob": torch.where(live, zt - lse.squeeze(1), 0.0), "entropy": torch.where(live, entropy, 0.0),
               "top_logprob": torch.where(live[:, None], ztop - lse, 0.0),
               "top_index": torch.where(live[:, None], top, -1)}
        if d is not None:
            glp, gh, gtop = d[0][i:i + step], d[1][i:i + step], d[2][i:i + step]
            g = (glp + gtop.sum(1))[:, None] + gh[:, None] * (z - log_s + entropy[:, None])
            dz = -p * g
            dz.scatter_add_(1, t.clamp_min(0)[:, None], glp[:, None])
            dz.scatter_add_(1, top, gtop)
            out["dlogits"] = (torch.where(live[:, None], dz, 0.0) / tau).to(x.dtype)
        parts.append(out)
    return {n: torch.cat([o[n] for o in parts]) for n in parts[0]}


# --------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "quantise":
            return _plain_quantise(state["x"], case["weight"])
        if kind == "linear":
            w = _values(_unpack(state["codes"]), state["exponents"], 32)
            return (_values(*_codes(state["x"], 1), 1) @ w.t()).to(state["x"].dtype)
        if kind == "train":
            return _plain_train(state["x"], state["w"], state["dy"])
        d = (state["d_logprob"], state["d_entropy"], state["d_top"]) if kind == "policy" else None
        return _plain_logprobs(case, state["logits"], state["target"], d)

    from flex_shard_b200.ops import logprobs, mxfp4, mxfp8
    from flex_shard_b200.quant import BlockwiseMxfp4Weight

    if kind == "quantise":
        x = state["x"]
        if not case["weight"]:
            return {"values": mxfp4.mx4_dequantize(*mxfp4.mx4_quantize_act(x))}
        q, e = mxfp4.mx4_quantize_weight(x)
        return {"values": mxfp4.mx4_dequantize(q, mxfp8.mx_expand_scales(e, *x.shape)), "exponents": e}
    if kind == "linear":
        with torch.no_grad():
            return mxfp4.mxfp4_linear(state["x"], None, state["codes"], state["scales"], None)
    if kind == "train":
        x, w = state["x"], state["w"]
        w4 = BlockwiseMxfp4Weight.from_float(w.detach())
        y = mxfp4.mxfp4_linear(x, w, w4.qdata, w4.scale, w4.dgrad_scale)
        dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    call = dict(temperature=case["temperature"], top_k=case["k"])
    if kind == "score":
        with torch.no_grad():
            return logprobs.token_logprobs(state["logits"], state["target"], **call)._asdict()
    out = logprobs.token_logprobs(state["logits"], state["target"], **call)
    heads = [out.logprob, out.entropy] + ([out.top_logprob] if case["k"] else [])
    grads = [state["d_logprob"], state["d_entropy"]] + ([state["d_top"]] if case["k"] else [])
    (dlogits,) = torch.autograd.grad(heads, state["logits"], grads)
    return {"logprob": out.logprob.detach(), "entropy": out.entropy.detach(), "top_logprob": out.top_logprob.detach(),
            "top_index": out.top_index, "dlogits": dlogits}


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "quantise":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * n + (-(-case["rows"] // 32) * case["cols"] // 32 if case["weight"] else 0), "flops": 2 * n}
    if kind in ("linear", "train"):
        T, N, K = case["T"], case["N"], case["K"]
        if kind == "linear":
            return {"bytes": 2 * T * (N + K) + N * K / 2 + N * K / 32, "flops": 2 * T * N * K}
        return {"bytes": 2 * 2 * (T * N + T * K + N * K), "flops": 6 * T * N * K}
    n = case["T"] * case["V"]
    size = 4 if case["dtype"] == "fp32" else 2
    small = case["T"] * (16 + 12 * case["k"])
    if kind == "score":
        return {"bytes": n * size + small, "flops": 4 * n}
    return {"bytes": 2 * n * size + 2 * small, "flops": 10 * n}


# --------------------------------------------------------------------------- 64 bits, from the definitions
def _two_to(e):
    """2^e in 64 bits, exactly (a device's pow may be off in the last bit, which decides ties)."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_scale(amax, top):
    """The smallest power of two s with amax / s <= top; 2^-127 at least."""
    e = torch.floor(torch.log2(amax.clamp_min(2.0 ** -149))) - 12
    for _ in range(16):
        e = torch.where(amax > top * _two_to(e), e + 1, e)
    return _two_to(e.clamp_min(-127))


def _exact_fp4(x, block):
    t = _groups(x.detach(), block).double()
    s = _exact_scale(t.abs().amax(dim=(1, 3), keepdim=True), 6.0)
    v = (t / s).abs()
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    q = torch.round(v / step) * step * torch.sign(t) * s            # round: ties to even multiples, as the codes are
    return q.view(-1, x.shape[1])[:x.shape[0]], s.view(s.shape[0], -1)


def _exact_fp8(x, dim):
    t = x.detach().double()
    t = t.t().contiguous() if dim == 0 else t
    t = t.view(t.shape[0], -1, 32)
    s = _exact_scale(t.abs().amax(-1, keepdim=True), 448.0)
    v = (t / s).abs()
    step = _two_to(torch.floor(torch.log2(v.clamp_min(2.0 ** -6))) - 3)
    q = (torch.round(v / step) * step * torch.sign(t) * s).view(t.shape[0], -1)
    return q.t() if dim == 0 else q


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantise":
        q, s = _exact_fp4(state["x"], 32 if case["weight"] else 1)
        return {"values": q, "exponents": torch.log2(s).add(127).round().to(torch.uint8)} if case["weight"] else {"values": q}
    if kind == "linear":
        c = _unpack(state["codes"]).long()
        half = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], device=GPU)[c & 7] * (1 - 2 * (c >> 3))
        s = _two_to(state["exponents"].long() - 128)
        w = half * s.repeat_interleave(32, 0)[:case["N"]].repeat_interleave(32, 1)
        del c, half, s
        return _exact_fp4(state["x"], 1)[0] @ w.t()
    if kind == "train":
        x, w, dy = state["x"], state["w"], state["dy"]
        w4 = _exact_fp4(w, 32)[0]
        if case["T"] % 128 == 0:
            dw = _exact_fp8(dy, 0).t() @ _exact_fp8(x, 0)
        else:
            dw = dy.double().t() @ x.detach().double()
        return {"y": _exact_fp4(x, 1)[0] @ w4.t(), "dx": _exact_fp8(dy, 1) @ w4, "dw": dw}
    T, V, k, tau = case["T"], case["V"], case["k"], case["temperature"]
    outs = []
    step = max(1, (1 << 25) // V)
    for i in range(0, T, step):
        x = state["logits"].detach()[i:i + step]
        t = state["target"][i:i + step]
        dead = t == -100
        z = x.double() / tau
        lp = torch.log_softmax(z, 1)
        finite = lp.masked_fill(lp == -math.inf, 0.0)
        H = -(lp.exp() * finite).sum(1)
        best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        at = t.masked_fill(dead, 0)[:, None]
        out = {"logprob": lp.gather(1, at)[:, 0].masked_fill(dead, 0), "entropy": H.masked_fill(dead, 0),
               "top_logprob": lp.gather(1, best).masked_fill(dead[:, None], 0),
               "top_index": best.masked_fill(dead[:, None], -1)}
        if kind == "policy":
            gl, ge, gt = (state[n][i:i + step].double() for n in ("d_logprob", "d_entropy", "d_top"))
            chosen = torch.zeros_like(lp).scatter_(1, at, gl[:, None]).scatter_add_(1, best, gt)
            p = lp.exp()
            dz = chosen - p * chosen.sum(1, keepdim=True) - ge[:, None] * p * (finite + H[:, None])
            out["dlogits"] = (dz / tau).masked_fill(dead[:, None], 0)
        outs.append(out)
    return {n: torch.cat([o[n] for o in outs]) for n in outs[0]}
