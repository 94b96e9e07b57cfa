"""MXFP4: e2m1 data (two codes a byte) with one power-of-two (e8m0) scale per 32 elements, quantisers and the
block-scaled tcgen05 GEMM (``kind::mxf4.block_scale``), with a linear autograd function.

Contract (the "round up" scaling rule of the MXFP8 operators, for a largest magnitude of 6): the scale of a group is the
smallest power of two ``s`` with ``amax / s <= 6``, stored as the byte ``log2(s) + 127`` (not below 0; 0 for an all-zero
group), ``q = e2m1(x / s)`` rounded to nearest with ties to even. A group that holds a NaN or an infinity gets the byte 255
(the format's NaN) and codes of 0: what it is multiplied into is NaN. Weights use 32x32 tiles, so that one set of tile
exponents serves the forward product and the input-gradient product; activations use 1x32 groups.

Codes are uint8 tensors ``[rows, cols / 2]``, the code of an even column in the low nibble. Scale tensors handed to the GEMM
are in the tensor core's block layout (``ops/mxfp8.py``). Columns are a multiple of 32. CPU tensors take a PyTorch
restatement of the same arithmetic.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import count_launch
from .gemm import gemm
from .mxfp8 import GROUP, MX_WGRAD, blocked_scale_numel, from_blocked, gemm_mxfp8, mx_quantize_act, mx_quantize_rows, to_blocked

FP8 = torch.float8_e4m3fn
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_KINDS = {FP8: 0, torch.bfloat16: 1, torch.float32: 2}
_declared = False


def _ensure():
    global _declared
    if not _declared:
        c = ctypes
        vp, i32, i64 = c.c_void_p, c.c_int, c.c_longlong
        _lib.declare("fsb_mx4_quant_act", [vp, vp, vp, i64, i32, i64, vp])
        _lib.declare("fsb_mx4_quant_weight", [vp, vp, vp, vp, vp, i32, i32, i64, vp])
        _lib.declare("fsb_mx4_expand", [vp, vp, vp, i64, i32, i64, i32, vp])
        _lib.declare("fsb_mxfp4_linear", [vp, i64, vp, i64, vp, vp, i64, vp, i64, i32, i32, i32, vp, vp])
        _lib.declare("fsb_mxfp4_linear_few", [i32, i32, i32])
        _lib.declare("fsb_mxfp4_linear_dx", [vp, i64, vp, i64, vp, vp, vp, i64, i32, i32, i32, vp, vp])
        _lib.declare("fsb_mxfp4_linear_dw", [vp, i64, vp, i64, vp, i32, vp, i64, i32, i32, i32, vp, vp])
        _lib.declare("fsb_gemm_mxfp4", [vp, vp, vp, vp, vp, i32, i32, i32, i64, i64, i64, i32, vp, vp])
        _declared = True


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    """Checked bf16 ``[rows, cols]`` with dense rows."""
    if x.dim() != 2 or x.shape[1] % GROUP or x.shape[1] == 0:
        raise ValueError(f"{what} must be a matrix whose columns are a multiple of {GROUP}, got {tuple(x.shape)}")
    if not x.is_floating_point():
        raise ValueError(f"{what} must be floating point, got {x.dtype}")
    x = x.detach()
    return x if (x.dtype == torch.bfloat16 and x.stride(1) == 1) else x.to(torch.bfloat16).contiguous()


def _check_operand(q: torch.Tensor, scales: torch.Tensor, what: str) -> None:
    shape = q.shape
    if len(shape) != 2 or q.dtype is not torch.uint8 or shape[1] % (GROUP // 2) or shape[1] == 0:
        raise ValueError(f"{what}: codes must be a uint8 matrix [rows, cols / 2] with cols a multiple of {GROUP}, got "
                         f"{q.dtype}{tuple(shape)}")
    _check_scales(scales, shape[0], 2 * shape[1], q.device, what)


def _check_scales(scales: torch.Tensor, rows: int, cols: int, device, what: str) -> None:
    need = (-(-rows // 128) * 128) * (-(-cols // 128) * 4)               # blocked_scale_numel(rows, cols)
    if scales.dtype is not torch.uint8 or scales.numel() < need or not scales.is_contiguous() or scales.device != device:
        raise ValueError(f"{what}: scales must be at least {need} contiguous uint8 bytes in block layout on the codes' device")


def _ld(t: torch.Tensor) -> int:
    """Row stride in elements; a single row has any stride."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


# --------------------------------------------------------------------------- restatement
def _exponent(amax: torch.Tensor) -> torch.Tensor:
    bits = amax.float().contiguous().view(torch.int32)
    e = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x400000).int()).clamp_min(0)
    return torch.where(bits >= 0x7F800000, torch.full_like(e, 255), e).to(torch.uint8)


def _scale(e: torch.Tensor) -> torch.Tensor:
    """``2^(e - 127)``, NaN for 255."""
    b = e.to(torch.int32)
    s = torch.where(b == 0, torch.full_like(b, 0x00400000), b << 23).view(torch.float32)
    return torch.where(b == 255, torch.full_like(s, float("nan")), s)


def _encode(t: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """Codes of fp32 values whose scale bytes ``e`` broadcast against them."""
    v = t * _scale((254 - e.to(torch.int32)).clamp_min(0).to(torch.uint8))
    v = torch.where(e == 255, torch.zeros_like(v), v)
    a = v.abs()
    # between the magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6; a midpoint goes to the even code
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return code | torch.signbit(v).to(torch.uint8) << 3


def _pack(codes: torch.Tensor) -> torch.Tensor:
    return codes[:, 0::2] | codes[:, 1::2] << 4


def _unpack(q: torch.Tensor) -> torch.Tensor:
    return torch.stack([q & 15, q >> 4], -1).reshape(q.shape[0], 2 * q.shape[1])


def mx4_quantize_act_ref(x: torch.Tensor):
    T, K = x.shape
    t = x.to(torch.bfloat16).float().reshape(T, K // GROUP, GROUP)
    e = _exponent(t.abs().amax(-1))
    return _pack(_encode(t, e[..., None]).view(T, K)), to_blocked(e)


def mx4_quantize_weight_ref(w: torch.Tensor):
    rows, cols = w.shape
    pad = torch.zeros(-(-rows // GROUP) * GROUP, cols, dtype=torch.float32, device=w.device)
    pad[:rows] = w.to(torch.bfloat16).float()
    t = pad.view(-1, GROUP, cols // GROUP, GROUP)
    e = _exponent(t.abs().amax(dim=(1, 3)))
    return _pack(_encode(t, e[:, None, :, None]).view(-1, cols)[:rows]).contiguous(), e


# --------------------------------------------------------------------------- quantisers
def mx4_quantize_act(x: torch.Tensor):
    """bf16 ``[T, K]`` -> (codes ``[T, K / 2]``, blocked uint8 scales), groups of 32 along the row. Other floating types
    are rounded to bf16 first."""
    x = _matrix(x, "the input")
    if not x.is_cuda:
        return mx4_quantize_act_ref(x)
    _ensure()
    T, K = x.shape
    q = torch.empty(T, K // 2, dtype=torch.uint8, device=x.device)
    s = torch.empty(blocked_scale_numel(T, K), dtype=torch.uint8, device=x.device)
    with _lib.device_of(x):
        rc = _lib.load().fsb_mx4_quant_act(x.data_ptr(), q.data_ptr(), s.data_ptr(), T, K, x.stride(0), _lib.stream_ptr(x.device))
    _lib.check(rc, "fsb_mx4_quant_act")
    count_launch(int(T > 0))
    return q, s


def _quantize_weight(w: torch.Tensor, layouts: bool):
    rows, cols = w.shape
    empty = lambda *n: torch.empty(*n, dtype=torch.uint8, device=w.device)  # noqa: E731
    q, e = empty(rows, cols // 2), empty(-(-rows // GROUP), cols // GROUP)
    fwd = empty(blocked_scale_numel(rows, cols)) if layouts else None
    dgrad = empty(blocked_scale_numel(cols, rows)) if layouts else None
    with _lib.device_of(w):
        rc = _lib.load().fsb_mx4_quant_weight(w.data_ptr(), q.data_ptr(), e.data_ptr(), fwd.data_ptr() if layouts else None,
                                              dgrad.data_ptr() if layouts else None, rows, cols, w.stride(0),
                                              _lib.stream_ptr(w.device))
    _lib.check(rc, "fsb_mx4_quant_weight")
    count_launch(int(rows > 0))
    return q, e, fwd, dgrad


def mx4_quantize_weight(w: torch.Tensor):
    """bf16 ``[rows, cols]`` -> (codes ``[rows, cols / 2]``, uint8 tile exponents ``[ceil(rows / 32), cols / 32]``)."""
    w = _matrix(w, "the weight")
    if not w.is_cuda:
        return mx4_quantize_weight_ref(w)
    _ensure()
    return _quantize_weight(w, False)[:2]


def mx4_quantize_weight_operands(w: torch.Tensor):
    """As ``mx4_quantize_weight`` with both operands' blocked scales from the same pass: (codes, tile exponents, scales of
    ``[rows, cols]`` for the forward product, scales of ``[cols, rows]`` for the input-gradient product)."""
    w = _matrix(w, "the weight")
    if not w.is_cuda:
        from .mxfp8 import mx_expand_scales

        q, e = mx4_quantize_weight_ref(w)
        return q, e, mx_expand_scales(e, *w.shape, False), mx_expand_scales(e, *w.shape, True)
    _ensure()
    return _quantize_weight(w, True)


def _expand(q: torch.Tensor, scales, dtype: torch.dtype) -> torch.Tensor:
    _ensure()
    T, K = q.shape[0], 2 * q.shape[1]
    if q.stride(1) != 1 or _ld(q) % 4 or q.data_ptr() % 4:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty(T, K, dtype=dtype, device=q.device)
    with _lib.device_of(q):
        rc = _lib.load().fsb_mx4_expand(q.data_ptr(), scales.data_ptr() if scales is not None else None, out.data_ptr(), T, K,
                                        _ld(q), _KINDS[dtype], _lib.stream_ptr(q.device))
    _lib.check(rc, "fsb_mx4_expand")
    count_launch(int(T > 0))
    return out


def mx4_dequantize(q: torch.Tensor, blocked: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Codes ``[rows, cols / 2]`` with blocked scales whose groups run along the columns -> ``[rows, cols]`` in bf16 or fp32
    (exact in both, but for what underflows)."""
    _check_operand(q, blocked, "mx4_dequantize")
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"mx4_dequantize gives bf16 or fp32, not {dtype}")
    if q.is_cuda:
        return _expand(q, blocked, dtype)
    c = _unpack(q).long()
    v = torch.tensor(_VALUES)[c & 7] * (1 - 2 * (c >> 3))
    e = from_blocked(blocked, q.shape[0], c.shape[1] // GROUP)
    return (v * _scale(e).repeat_interleave(GROUP, 1)).to(dtype)


def mx4_to_e4m3(q: torch.Tensor) -> torch.Tensor:
    """The codes' values, without scales, as e4m3 ``[rows, cols]``: the same operand for the 8-bit products (exact)."""
    if q.dim() != 2 or q.dtype != torch.uint8 or q.shape[1] % (GROUP // 2) or q.shape[1] == 0:
        raise ValueError(f"codes must be a uint8 matrix [rows, cols / 2] with cols a multiple of {GROUP}")
    if q.is_cuda:
        return _expand(q, None, FP8)
    c = _unpack(q).long()
    return (torch.tensor(_VALUES)[c & 7] * (1 - 2 * (c >> 3))).to(FP8)


# --------------------------------------------------------------------------- GEMM
def gemm_mxfp4(aq, sfa, bq, sfb, *, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``out[M, N] = (A * 2^sfa) . (B * 2^sfb)^T`` for codes ``aq [M, K / 2]`` and ``bq [N, K / 2]`` with blocked scales,
    accumulated in fp32, rounded once (bf16) or not (fp32)."""
    _check_operand(aq, sfa, "gemm_mxfp4: left operand")
    _check_operand(bq, sfb, "gemm_mxfp4: right operand")
    if aq.shape[1] != bq.shape[1] or aq.device != bq.device:
        raise ValueError(f"gemm_mxfp4: operands {tuple(aq.shape)} and {tuple(bq.shape)} on {aq.device} and {bq.device}")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"gemm_mxfp4 gives bf16 or fp32, not {out_dtype}")
    M, N, K = aq.shape[0], bq.shape[0], 2 * aq.shape[1]
    if not aq.is_cuda:
        return (mx4_dequantize(aq, sfa, torch.float32) @ mx4_dequantize(bq, sfb, torch.float32).t()).to(out_dtype)
    out = torch.empty(M, N, dtype=out_dtype, device=aq.device)
    if M == 0 or N == 0:
        return out
    _ensure()
    aq, bq = (t if t.stride(1) == 1 and _ld(t) % 16 == 0 and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
              for t in (aq, bq))
    sfa, sfb = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (sfa, sfb))
    status = _lib.status_word(aq.device)
    with _lib.device_of(aq):
        rc = _lib.load().fsb_gemm_mxfp4(aq.data_ptr(), sfa.data_ptr(), bq.data_ptr(), sfb.data_ptr(), out.data_ptr(), M, N, K,
                                        _ld(aq), _ld(bq), N, int(out_dtype == torch.float32),
                                        status.data_ptr(), _lib.stream_ptr(aq.device))
    _lib.check(rc, "fsb_gemm_mxfp4")
    count_launch()
    return out


@functools.lru_cache(maxsize=1024)
def _one_launch(T: int, N: int, K: int) -> bool:
    """Whether the linear quantises its rows inside the product and needs no scratch (a rule on the sizes alone)."""
    return bool(_lib.load().fsb_mxfp4_linear_few(T, N, K))


def _product_with(x2, wq, fwd_scale):
    """``[T, K]`` rows times the quantised weight: the forward pass of ``mxfp4_linear``."""
    T, K = x2.shape
    N = wq.shape[0]
    if not x2.is_cuda:
        return gemm_mxfp4(*mx4_quantize_act(x2), wq, fwd_scale)
    out = x2.new_empty(T, N)
    if T == 0 or N == 0:
        return out
    _ensure()
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    ldx, ldw = x2.stride(0) if T > 1 else K, wq.stride(0) if N > 1 else K // 2
    if wq.stride(1) != 1 or ldw % 16 or wq.data_ptr() % 16:
        wq = wq.clone(memory_format=torch.contiguous_format)
        ldw = K // 2
    if fwd_scale.data_ptr() % 16:
        fwd_scale = fwd_scale.clone()
    scratch, size = None, 0
    if T > 16 or not _one_launch(T, N, K):
        size = T * (K // 2) + blocked_scale_numel(T, K)     # codes, scales
        scratch = torch.empty(size, dtype=torch.uint8, device=x2.device)
    with _lib.device_of(x2):
        rc = _lib.load().fsb_mxfp4_linear(x2.data_ptr(), ldx, wq.data_ptr(), ldw, fwd_scale.data_ptr(), out.data_ptr(), N,
                                          None if scratch is None else scratch.data_ptr(), size, T, N, K,
                                          _lib.status_word(x2.device).data_ptr(), _lib.stream_ptr(x2.device))
    _lib.check(rc, "fsb_mxfp4_linear")
    count_launch(1 if scratch is None else 2)
    return out


def _input_gradient(dy2, wq, dgrad_scale):
    """``dy2 [T, N]`` in MXFP8 groups along N times the codes' own values."""
    (T, N), K = dy2.shape, 2 * wq.shape[1]
    if not dy2.is_cuda:
        return gemm_mxfp8(*mx_quantize_act(dy2), mx4_to_e4m3(wq), dgrad_scale, b_t=True)
    _ensure()
    if wq.stride(1) != 1 or wq.stride(0) % 4 or wq.data_ptr() % 4:
        wq = wq.clone(memory_format=torch.contiguous_format)
    if dgrad_scale.data_ptr() % 16:
        dgrad_scale = dgrad_scale.clone()
    dx = dy2.new_empty(T, K)
    size = T * N + N * K + blocked_scale_numel(T, N)
    scratch = torch.empty(size, dtype=torch.uint8, device=dy2.device)
    with _lib.device_of(dy2):
        rc = _lib.load().fsb_mxfp4_linear_dx(dy2.data_ptr(), N, wq.data_ptr(), wq.stride(0), dgrad_scale.data_ptr(), dx.data_ptr(),
                                             scratch.data_ptr(), size, T, N, K, _lib.status_word(dy2.device).data_ptr(),
                                             _lib.stream_ptr(dy2.device))
    _lib.check(rc, "fsb_mxfp4_linear_dx")
    count_launch(3)
    return dx


def _input_gradient_bf16(dy2, wq, fwd_scale):
    """The same in bf16, for any N and K: the codes' values times their scales are bf16 numbers. N is padded to the product's 8."""
    w, pad = mx4_dequantize(wq, fwd_scale), -wq.shape[0] % 8
    if pad:
        w, dy2 = torch.nn.functional.pad(w, (0, 0, 0, pad)), torch.nn.functional.pad(dy2, (0, pad))
    return gemm(dy2, w, b_t=True)


def _weight_gradient(dy2, x2, dtype):
    """``dy2^T x2`` with both operands in MXFP8 groups along the rows (all dims multiples of 128)."""
    (T, N), K = dy2.shape, x2.shape[1]
    if not dy2.is_cuda:
        return gemm_mxfp8(*mx_quantize_rows(dy2), *mx_quantize_rows(x2), a_t=True, b_t=True, out_dtype=dtype)
    _ensure()
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    dw = torch.empty(N, K, dtype=dtype, device=dy2.device)
    size = (T + T // 32) * (N + K)
    scratch = torch.empty(size, dtype=torch.uint8, device=dy2.device)
    with _lib.device_of(dy2):
        rc = _lib.load().fsb_mxfp4_linear_dw(dy2.data_ptr(), N, x2.data_ptr(), x2.stride(0), dw.data_ptr(), int(dtype == torch.float32),
                                             scratch.data_ptr(), size, T, N, K, _lib.status_word(dy2.device).data_ptr(),
                                             _lib.stream_ptr(dy2.device))
    _lib.check(rc, "fsb_mxfp4_linear_dw")
    count_launch(3)
    return dw


class _Mxfp4Linear(torch.autograd.Function):
    """y = x W^T in 4 bits; gradients in 8 bits with the 4-bit weights' own values (quantisation counts as the identity)."""

    @staticmethod
    def forward(ctx, x, weight, wq, fwd_scale, dgrad_scale):
        x2 = x.reshape(-1, x.shape[-1])
        ctx.save_for_backward(x2, wq, fwd_scale, dgrad_scale)
        ctx.xshape = x.shape
        ctx.weight = weight
        return _product_with(x2, wq, fwd_scale).view(*x.shape[:-1], wq.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, wq, fwd_scale, dgrad_scale = ctx.saved_tensors
        weight = ctx.weight
        N, K = wq.shape[0], x2.shape[1]
        dy2 = dy.reshape(-1, N).contiguous()
        T = dy2.shape[0]
        dx = dw = None
        if ctx.needs_input_grad[0]:
            if T == 0:
                dx = torch.zeros(ctx.xshape, dtype=x2.dtype, device=x2.device)
            elif N % 128 or K % 128:
                dx = _input_gradient_bf16(dy2, wq, fwd_scale).view(ctx.xshape)
            else:
                dx = _input_gradient(dy2, wq, dgrad_scale).view(ctx.xshape)
        if ctx.needs_input_grad[1]:
            main = getattr(weight, "main_grad", None)
            gd = getattr(weight, "grad_dtype", None) or torch.bfloat16
            gd = gd if gd in (torch.bfloat16, torch.float32) else torch.bfloat16
            if main is not None and main.dtype in (torch.float32, torch.bfloat16):
                if T > 0:
                    gemm(dy2, x2, a_t=True, b_t=True, out=main, accumulate=bool(getattr(weight, "main_grad_written", False)))
                    weight.main_grad_written = True
            elif T == 0:
                dw = torch.zeros(N, K, dtype=gd, device=x2.device)
            elif MX_WGRAD and T % 128 == 0 and N % 128 == 0 and K % 128 == 0:
                dw = _weight_gradient(dy2, x2, gd)
            else:
                dw = gemm(dy2, x2, a_t=True, b_t=True, out_dtype=gd)
        return dx, dw, None, None, None


def mxfp4_linear(x, weight, wq, fwd_scale, dgrad_scale, *, bf16_input_gradient: bool = False):
    """``x @ W.T`` for bf16 ``x [..., K]`` (K a multiple of 32) and a weight given as MXFP4 codes ``wq [N, K / 2]`` with the
    blocked scales of the operands ``[N, K]`` (forward) and ``[K, N]`` (input gradient; may be ``None`` where no gradient
    of ``x`` is asked for). ``weight`` is the logical parameter that receives the weight gradient, or ``None`` for a frozen
    weight.

    The gradient of ``x`` is an 8-bit product with the 4-bit weight's own values and needs N and K in multiples of 128; with
    ``bf16_input_gradient`` other sizes take a bf16 product with the same values instead of a refusal (as ``linear`` does for
    frozen weights). The weight's gradient is an 8-bit product where the number of rows, N and K are multiples of 128 and the
    parameter has no gradient bucket, else a bf16 one, and needs N and K in multiples of 8."""
    if x.dtype != torch.bfloat16:
        raise ValueError(f"mxfp4_linear takes bf16 inputs, got {x.dtype}")
    _check_operand(wq, fwd_scale, "mxfp4_linear")
    N, K = wq.shape[0], 2 * wq.shape[1]
    if x.dim() < 1 or x.shape[-1] != K or x.device != wq.device:
        raise ValueError(f"mxfp4_linear: input {tuple(x.shape)} on {x.device} does not match codes {tuple(wq.shape)} ([N, K / 2]) on "
                         f"{wq.device}")
    needs_x = x.requires_grad and torch.is_grad_enabled()
    needs_w = weight is not None and weight.requires_grad and torch.is_grad_enabled()
    if not (needs_x or needs_w) and _lib.plain(x) and forward_ad._current_level < 0:
        y = _product_with(x if x.dim() == 2 else x.reshape(-1, K), wq, fwd_scale)       # nothing to differentiate
        return y if x.dim() == 2 else y.view(*x.shape[:-1], N)
    if needs_x or needs_w:
        if needs_x and not (bf16_input_gradient and (N % 128 or K % 128)):
            if N % 128 or K % 128:
                raise ValueError(f"the input gradient of mxfp4_linear needs dims that are multiples of 128, got {N} x {K}")
            if dgrad_scale is None:
                raise ValueError("the input gradient of mxfp4_linear needs the scales of the transposed weight (dgrad_scale)")
            _check_scales(dgrad_scale, K, N, wq.device, "mxfp4_linear (dgrad_scale)")
        if needs_w and (N % 8 or K % 8):
            raise ValueError(f"the weight gradient of mxfp4_linear needs dims that are multiples of 8, got {N} x {K}")
    return _Mxfp4Linear.apply(x, weight, wq, fwd_scale, dgrad_scale)
