"""Low-rank adapters beside a shared projection: of one model that is tuned while its weights stay frozen (`fp8_block_linear` gives these no
gradient), or of many requests served together, each row with its own.

Row t with adapter l = index[t]: out[t] = base[t] + s_l (x[t] A_l^T) B_l^T.  Rows are not sorted and adapters not gathered; a row without an
adapter is its base.  The reference has no adapters."""
from __future__ import annotations

import torch

from . import _lib as L

__all__ = ["lora_linear"]

MAX_RANK, MAX_ADAPTERS = 128, 65536


def _rows(t):
    """t as rows that the kernels read in place where they can: neighbouring values, at multiples of 16 bytes"""
    t = t.reshape(-1, t.shape[-1])
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0 or t.numel() == 0:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _aligned(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _Lora(torch.autograd.Function):
    """base (..., N) or zeros, plus x (..., K) through each row's adapter of a (L,R,K), b (L,N,R).  Plain calls take its compiled form (csrc/fast.cpp)."""

    @staticmethod
    def forward(ctx, x, a, b, base, index, scales, scale):
        (n, R, K), N, dev, lib = a.shape, b.shape[1], x.device, L.lib()
        ctx.types = a.dtype, b.dtype
        x2, a, b = _rows(x), _aligned(a.to(torch.bfloat16)), _aligned(b.to(torch.bfloat16))
        base2 = None if base is None else _rows(base)
        index = None if index is None else index.contiguous()
        T, keep = x2.shape[0], any(ctx.needs_input_grad[:3])
        with L.on_device_of(x):
            out = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=dev)
            ws = L.workspace(lib.b200moe_lora_fwd_ws_bytes(T, R, n, int(keep)), dev)
            if T:
                L.check(lib.b200moe_lora_forward(x2.data_ptr(), x2.stride(0), a.data_ptr(), b.data_ptr(), L.ptr(index), 0 if index is None else
                                                 index.element_size(), L.ptr(scales), scale, L.ptr(base2), 0 if base2 is None else base2.stride(0), T, K, N,
                                                 R, n, int(keep), ws.data_ptr(), out.data_ptr(), L.status_word(dev).data_ptr(), L.stream_of(x)))
        ctx.scale, ctx.has_index = scale, index is not None
        if keep:
            ctx.save_for_backward(x, a, b, scales, ws)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        need_x, need_a, need_b, need_base = ctx.needs_input_grad[:4]
        gx = ga = gb = None
        if need_x or need_a or need_b:
            x, a, b, scales, ws = ctx.saved_tensors
            (n, R, K), N, dev, lib, x2 = a.shape, b.shape[1], a.device, L.lib(), _rows(x)
            T, wide = x2.shape[0], ctx.types[0] == torch.float32
            with L.on_device_of(x):
                go = _aligned(grad.to(torch.bfloat16))
                gx = torch.empty(x.shape, dtype=torch.bfloat16, device=dev) if need_x else None
                ga = torch.empty(a.shape, dtype=ctx.types[0], device=dev) if need_a else None
                gb = torch.empty(b.shape, dtype=ctx.types[1], device=dev) if need_b else None
                if T:
                    tmp = L.workspace(lib.b200moe_lora_bwd_ws_bytes(T, K, N, R, n), dev)
                    L.check(lib.b200moe_lora_backward(go.data_ptr(), x2.data_ptr(), x2.stride(0), a.data_ptr(), b.data_ptr(), int(ctx.has_index),
                                                      L.ptr(scales), ctx.scale, T, K, N, R, n, ws.data_ptr(), tmp.data_ptr(), L.ptr(gx), L.ptr(ga),
                                                      L.ptr(gb), int(wide), L.status_word(dev).data_ptr(), L.stream_of(x)))
                else:
                    ga, gb = (None if t is None else t.zero_() for t in (ga, gb))
        return gx, ga, gb, grad if need_base else None, None, None, None


def lora_linear(x, lora_a, lora_b, index=None, scaling=1.0, base=None):
    """x (..., K) bf16 through the low-rank adapters lora_a (L,R,K) and lora_b (L,N,R), added to base (..., N) bf16 (None: to zero) -> (..., N) bf16:
    out[t] = base[t] + s_l (x[t] A_l^T) B_l^T with l = index[t].

    index: int32 or int64 of x's leading shape; a negative one is a row without an adapter, whose out is its base (one of L or more too, and it
    raises the status word).  None: one adapter (L = 1) for every row.  scaling: a number, or fp32 (L,).  K and N multiples of 8, the rank R of 8 up to
    128 (smaller ones of a stack are padded with zeros).  Adapters are bf16, or fp32 that is rounded to it and gets fp32 gradients.  Sums are fp32,
    x A^T goes on in 16 bits or more (two bf16 numbers) and the result is rounded once.  Rows and adapters do not mix: NaN or an infinity in one stays
    there (an infinity in lora_b may come out as NaN).  Differentiable in x, lora_a, lora_b and base; scaling takes no gradient."""
    fast = L.fast() if x.is_cuda else None
    if fast is not None:
        wide = isinstance(scaling, torch.Tensor)
        out = fast.lora_linear(x, lora_a, lora_b, index, scaling if wide else None, 1.0 if wide else scaling, base, L.status_word(x.device))
        if out is not None:
            return out
    if torch.is_autocast_enabled("cuda") and x.is_floating_point():
        dt = torch.get_autocast_dtype("cuda")
        x, base = x.to(dt), None if base is None else base.to(dt)
    L.require_cuda_bf16("x", x)
    L.require(lora_a.dim() == 3 and lora_b.dim() == 3, "lora_a must be (L,R,K) and lora_b (L,N,R)")
    (n, R, K), (n2, N, R2), dev = lora_a.shape, lora_b.shape, x.device
    L.require(n == n2 and R == R2, f"lora_a (L,R,K) and lora_b (L,N,R) must agree, got {tuple(lora_a.shape)} and {tuple(lora_b.shape)}")
    L.require(lora_a.dtype == lora_b.dtype and lora_a.dtype in (torch.bfloat16, torch.float32),
              f"lora_a and lora_b must both be bfloat16 or both float32, got {lora_a.dtype} and {lora_b.dtype}")
    L.require(lora_a.device == dev and lora_b.device == dev, "lora_a and lora_b must be on x's device")
    L.require(x.dim() >= 1 and x.shape[-1] == K, f"x must be (..., {K}), got {tuple(x.shape)}")
    L.require(1 <= n <= MAX_ADAPTERS, f"1 to {MAX_ADAPTERS} adapters are supported, got {n}")
    L.require(K > 0 and N > 0 and K % 8 == 0 and N % 8 == 0, f"K and N must be positive multiples of 8, got {K} and {N}")
    L.require(8 <= R <= MAX_RANK and R % 8 == 0, f"the rank must be a multiple of 8 up to {MAX_RANK}, got {R}")
    if index is None:
        L.require(n == 1, f"without an index there is one adapter, got {n}")
    else:
        L.require(index.device == dev and index.dtype in (torch.int32, torch.int64) and index.shape == x.shape[:-1],
                  f"index must be int32 or int64 {tuple(x.shape[:-1])} on x's device, got {index.dtype} {tuple(index.shape)}")
    scales = None
    if isinstance(scaling, torch.Tensor):
        L.require(scaling.device == dev and scaling.dtype == torch.float32 and tuple(scaling.shape) == (n,),
                  f"scaling must be a number or float32 ({n},) on x's device, got {scaling.dtype} {tuple(scaling.shape)}")
        L.require(not (torch.is_grad_enabled() and scaling.requires_grad), "scaling takes no gradient: scaling.detach()")
        scales, scaling = scaling.contiguous(), 1.0
    if base is not None:
        L.require(base.device == dev and base.dtype == torch.bfloat16 and base.shape == (*x.shape[:-1], N),
                  f"base must be bfloat16 {(*x.shape[:-1], N)} on x's device, got {base.dtype} {tuple(base.shape)}")
    return _Lora.apply(x, lora_a, lora_b, base, index, scales, float(scaling))
