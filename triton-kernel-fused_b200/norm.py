"""Root-mean-square norm with the residual's addition, and its rows in 8 bits for the products over block-scaled weights.

h = x + residual in x's type, y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.  The norm is of h as it goes on, rounded, so that
the backward computes the gradient of what the forward gave; sums are fp32, and codes are made from y before it is rounded.  One pass over
memory each way.  The reference has no norm of its own: its models put one before the layer that is built here."""
from __future__ import annotations

import torch

from . import _lib as L
from . import ops

__all__ = ["rms_norm", "rms_norm_fp8_block"]

BLOCK = 128
MAX_K = 16384


def _rows(t, K):
    """t as rows of K, in place where they lie at one distance"""
    t = t.reshape(-1, K)
    return t if t.stride(1) == 1 and t.stride(0) >= K or t.numel() == 0 else t.contiguous()


class _RmsNorm(torch.autograd.Function):
    """(y, h, codes, scales [block][row]) of x (..., K), each None that is not asked for or (h) has no residual; scales lie at a pitch that the
    products read without a copy.  Plain calls take its compiled form (csrc/fast.cpp)."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, want_y, want_codes):
        K, dev, lib = x.shape[-1], x.device, L.lib()
        x2, r2 = _rows(x, K), None if residual is None else _rows(residual, K)
        weight, N = weight.contiguous(), x2.shape[0]
        with L.on_device_of(x):
            y = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_y else None
            h = torch.empty(x.shape, dtype=x.dtype, device=dev) if residual is not None else None
            q = scale = None
            pitch = -(-N // BLOCK) * BLOCK
            if want_codes:
                q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
                scale = torch.empty(-(-K // BLOCK), pitch, dtype=torch.float32, device=dev)
            if N:
                L.check(lib.b200moe_rms_norm_fwd(x2.data_ptr(), x2.stride(0), L.ptr(r2), 0 if r2 is None else r2.stride(0), ops._LOGITS[x.dtype],
                                                 weight.data_ptr(), ops._LOGITS[weight.dtype], N, K, eps, L.ptr(y), L.ptr(h), L.ptr(q), L.ptr(scale),
                                                 pitch, L.status_word(dev).data_ptr(), L.stream_of(x)))
        ctx.save_for_backward(x if h is None else h, weight)
        ctx.eps = eps
        if want_codes:
            ctx.mark_non_differentiable(q, scale)
        ctx.set_materialize_grads(False)
        return y, h, q, scale

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_h, grad_q, grad_scale):
        h, weight = ctx.saved_tensors
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        if grad_y is None:       # the stream alone was used
            return grad_h if need_x else None, grad_h if need_r else None, None, None, None, None
        K, dev, lib = h.shape[-1], h.device, L.lib()
        h2, grad_y = _rows(h, K), grad_y.contiguous()
        grad_h = None if grad_h is None else grad_h.contiguous()
        N = h2.shape[0]
        with L.on_device_of(h):
            gx = torch.empty(h.shape, dtype=h.dtype, device=dev) if need_x or need_r else None
            gw = torch.empty_like(weight) if need_w else None
            ws = L.workspace(lib.b200moe_rms_norm_bwd_ws_bytes(N, K), dev) if need_w else None
            if N or need_w:
                L.check(lib.b200moe_rms_norm_bwd(grad_y.data_ptr(), L.ptr(grad_h), h2.data_ptr(), max(h2.stride(0), K), ops._LOGITS[h.dtype],
                                                 weight.data_ptr(), ops._LOGITS[weight.dtype], N, K, ctx.eps, L.ptr(ws), L.ptr(gx), L.ptr(gw),
                                                 L.status_word(dev).data_ptr(), L.stream_of(h)))
        return gx if need_x else None, gx if need_r else None, gw, None, None, None


def _check(x, weight, residual, eps, codes):
    L.require(x.is_cuda, "x must be a CUDA tensor (this package has no CPU path)")
    L.require(x.dtype in ops._LOGITS, f"x must be bfloat16, float16 or float32, got {x.dtype}")
    L.require(x.dim() >= 1 and 1 <= x.shape[-1] <= MAX_K, f"the last dimension of x must be 1 to {MAX_K}, x is {tuple(x.shape)}")
    L.require(not codes or x.shape[-1] % 8 == 0, f"codes want a last dimension that is a multiple of 8, x is {tuple(x.shape)}")
    L.require(weight.device == x.device and weight.shape == x.shape[-1:], f"weight must be ({x.shape[-1]},) on x's device, got {tuple(weight.shape)}")
    L.require(weight.dtype in (x.dtype, torch.float32), f"weight must be {x.dtype} or float32, got {weight.dtype}")
    if residual is not None:
        L.require(residual.device == x.device and residual.dtype == x.dtype and residual.shape == x.shape,
                  f"residual must be {x.dtype} {tuple(x.shape)} on x's device, got {residual.dtype} {tuple(residual.shape)}")
    eps = float(eps)
    L.require(0.0 <= eps <= torch.finfo(torch.float32).max, f"eps = {eps} must be finite in fp32 and not negative")
    return eps


def rms_norm(x, weight, residual=None, eps=1e-6):
    """x (..., K) bf16, fp16 or fp32, weight (K,) of x's type or fp32, residual like x -> y, or (y, h) with a residual: h = x + residual (rounded to
    x's type) and y = h / sqrt(mean(h^2) + eps) * weight.  K up to 16384; rows may lie at any distance.  Differentiable in x, residual and
    weight, through y and h."""
    fast = L.fast() if x.is_cuda else None
    if fast is not None:
        res = fast.rms_norm(x, weight, residual, eps, True, False, L.status_word(x.device))
        if res is not None:
            return res[0] if residual is None else res[:2]
    eps = _check(x, weight, residual, eps, False)
    y, h, _, _ = _RmsNorm.apply(x, residual, weight, eps, True, False)
    return y if residual is None else (y, h)


def rms_norm_fp8_block(x, weight, residual=None, eps=1e-6, return_norm=False):
    """`rms_norm` whose rows leave as the block-scaled products read them: (codes float8_e4m3fn (..., K), scales fp32 (..., ceil(K/128))[, y][, h]),
    the values being code * scale; y where return_norm, h where there is a residual.  K a multiple of 8.  Codes are made from y before its
    rounding (`fp8_block_quantize(y)` rounds twice) and are the nearest up to fp32's roundings of y and of the scale: a value in the middle between two
    codes may take either.  `fp8_block_linear(y, w, s, quantized=(codes, scales))` takes them; they carry no gradient,
    y and h do."""
    fast = L.fast() if x.is_cuda else None
    res = None if fast is None else fast.rms_norm(x, weight, residual, eps, bool(return_norm), True, L.status_word(x.device))
    if res is not None:
        y, h, q, scale = res
        return (q, scale) + ((y,) if return_norm else ()) + ((h,) if residual is not None else ())
    eps = _check(x, weight, residual, eps, True)
    y, h, q, scale = _RmsNorm.apply(x, residual, weight, eps, bool(return_norm), True)
    scale = scale[:, : x.numel() // x.shape[-1]].t().reshape(*x.shape[:-1], scale.shape[0])
    return (q, scale) + ((y,) if return_norm else ()) + ((h,) if residual is not None else ())
