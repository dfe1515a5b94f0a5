"""Products in 8-bit floating point with a scale per block of 128: e4m3 codes, fp32 scales, as 8-bit checkpoints hold them.

Weights carry one scale per 128 x 128 values, (..., ceil(N/128), ceil(K/128)); rows of activations are quantised on the way, one scale
per 128 values, nearest e4m3 to 448 x / max |x|.  Every block of 128 is summed in fp32 by the tensor cores, scaled, and added in fp32;
a product is rounded to bf16 once.  (So is what `moe_fp8_block` gives at few rows an expert; from 40 rows on an expert's results are bf16 before they
are weighted and summed, as in `moe`.)  MXFP8 (`moe_mxfp8`) is the other 8-bit format here: power-of-two scales per 32 values, bf16
masters, training.  These weights have no master: they are frozen, so `fp8_block_linear` gives the gradient of its input alone,
and `moe_fp8_block` serves.  The reference has no 8-bit path."""
from __future__ import annotations

import torch

from . import _lib as L

__all__ = ["fp8_block_linear", "fp8_block_quantize", "fp8_block_quantize_weight", "moe_fp8_block"]

BLOCK = 128


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _weight(name, w, scale, device, dim):
    """Codes and scales as the kernels read them: contiguous, 16-byte aligned."""
    L.require(w.dtype == torch.float8_e4m3fn and w.dim() == dim, f"{name} must be a float8_e4m3fn tensor of {dim} dimensions")
    L.require(w.device == device and scale.device == device, f"{name} and its scale must be on the input's device")
    L.require(not (torch.is_grad_enabled() and (w.requires_grad or scale.requires_grad)),
              f"{name} and its scale are frozen, they take no gradient: requires_grad_(False) on both, or torch.no_grad() around the call")
    want = (*w.shape[:-2], _blocks(w.shape[-2]), _blocks(w.shape[-1]))
    L.require(scale.dtype == torch.float32 and tuple(scale.shape) == want, f"the scale of {name} must be float32 {want}, got "
              f"{scale.dtype} {tuple(scale.shape)}")
    return w.contiguous(), scale.contiguous()


def _aligned(t):
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _Frozen(torch.autograd.Function):
    """Functions whose results take no gradient.  They are Functions all the same: a tracer records them as calls, where it would otherwise
    record nothing but the allocation of their results, and a forward-mode gradient, which they cannot carry on, is refused."""

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("the products of frozen 8-bit weights and their quantisers have no backward (moe and moe_mxfp8 train)")


class _Quantize(_Frozen):
    """(codes (N,K), scales (ceil(K/128), N)) of rows (N,K)"""

    @staticmethod
    def forward(ctx, rows):
        (N, K), rows = rows.shape, _aligned(rows)
        with L.on_device_of(rows):
            q = torch.empty(rows.shape, dtype=torch.float8_e4m3fn, device=rows.device)
            scale = torch.empty(_blocks(K), N, dtype=torch.float32, device=rows.device)
            if N:
                L.check(L.lib().b200moe_fp8_block_quant(rows.data_ptr(), N, K, q.data_ptr(), K, scale.data_ptr(), N, L.stream_of(rows)))
        ctx.mark_non_differentiable(q, scale)
        return q, scale


class _QuantizeWeight(_Frozen):
    """(codes, scales) of matrices (...,N,K)"""

    @staticmethod
    def forward(ctx, w):
        (N, K), w = w.shape[-2:], _aligned(w)
        with L.on_device_of(w):
            q = torch.empty(w.shape, dtype=torch.float8_e4m3fn, device=w.device)
            scale = torch.empty(*w.shape[:-2], _blocks(N), _blocks(K), dtype=torch.float32, device=w.device)
            L.check(L.lib().b200moe_fp8_block_quant_weight(w.data_ptr(), w.numel() // (N * K), N, K, q.data_ptr(), scale.data_ptr(),
                                                           L.stream_of(w)))
        ctx.mark_non_differentiable(q, scale)
        return q, scale


def fp8_block_quantize(x):
    """bf16 (..., K), K a multiple of 8 -> (codes float8_e4m3fn (..., K), scales fp32 (..., ceil(K/128))), the values being code * scale."""
    L.require_cuda_bf16("x", x)
    L.require(x.dim() >= 1 and x.shape[-1] > 0 and x.shape[-1] % 8 == 0, "the last dimension of x must be a positive multiple of 8")
    q, scale = _Quantize.apply(x.reshape(-1, x.shape[-1]).contiguous())
    return q.view(x.shape), scale.t().reshape(*x.shape[:-1], _blocks(x.shape[-1]))


def fp8_block_quantize_weight(w):
    """bf16 (..., N, K), K a multiple of 8 -> (codes float8_e4m3fn (..., N, K), scales fp32 (..., ceil(N/128), ceil(K/128)))."""
    L.require_cuda_bf16("w", w)
    L.require(w.dim() >= 2 and w.numel() > 0 and w.shape[-1] % 8 == 0, "w must be (..., N, K) with K a positive multiple of 8")
    return _QuantizeWeight.apply(w.contiguous())


def _product(x, w, scale, transposed):
    """x (M,K) * w (N,K)^T, or x (M,N) * w"""
    (N, K), M, dev = w.shape, x.shape[0], x.device
    lib = L.lib()
    with L.on_device_of(x):
        out = torch.empty(M, K if transposed else N, dtype=torch.bfloat16, device=dev)
        if M:
            ws = L.workspace(lib.b200moe_fp8_block_linear_ws_bytes(M, N if transposed else K), dev)
            L.check(lib.b200moe_fp8_block_linear(x.data_ptr(), w.data_ptr(), scale.data_ptr(), M, N, K, int(transposed), ws.data_ptr(),
                                                 out.data_ptr(), L.status_word(dev).data_ptr(), L.stream_of(x)))
    return out


class _Fp8BlockLinear(torch.autograd.Function):
    """x (M,K) through frozen weights; the gradient of x is the product of its own gradient, quantised like x, with the same codes.  Plain
    calls take its compiled form (csrc/fast.cpp)."""

    @staticmethod
    def forward(ctx, x, w, scale):
        x, w = _aligned(x), _aligned(w)      # in here: a tracer would keep the choice it saw
        ctx.save_for_backward(w, scale)
        return _product(x, w, scale, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        w, scale = ctx.saved_tensors
        return _product(_aligned(grad.to(torch.bfloat16).contiguous()), w, scale, True), None, None


def fp8_block_linear(x, weight, weight_scale):
    """x (..., K) bf16 times weight (N, K) float8_e4m3fn with weight_scale (ceil(N/128), ceil(K/128)) fp32 -> (..., N) bf16.
    N a multiple of 8, K of 16.  Differentiable in x (its gradient is quantised along N); the weights are frozen: one that
    requires a gradient is refused in grad mode."""
    fast = L.fast() if x.is_cuda else None
    if fast is not None:
        out = fast.fp8_block_linear(x, weight, weight_scale, L.status_word(x.device))
        if out is not None:
            return out
    if torch.is_autocast_enabled("cuda") and x.is_floating_point():
        x = x.to(torch.get_autocast_dtype("cuda"))
    L.require_cuda_bf16("x", x)
    w, scale = _weight("weight", weight, weight_scale, x.device, 2)
    N, K = w.shape
    L.require(x.dim() >= 1 and x.shape[-1] == K, f"x must be (..., {K}), got {tuple(x.shape)}")
    L.require(N % 8 == 0 and K % 16 == 0 and N > 0 and K > 0, f"weight must be (N, K) with N a multiple of 8 and K of 16, got ({N}, {K})")
    out = _Fp8BlockLinear.apply(x.reshape(-1, K).contiguous(), w, scale)
    return out if x.dim() == 2 else out.view(*x.shape[:-1], N)


class _Experts(_Frozen):
    """`moe_fp8_block` on checked and contiguous tensors."""

    @staticmethod
    def forward(ctx, hidden, idx, w, gu, gs, dn, ds):
        (T, H), (E, twoI, _), k, dev, lib = hidden.shape, gu.shape, idx.shape[1], hidden.device, L.lib()
        I = twoI // 2
        hidden, gu, dn = _aligned(hidden), _aligned(gu), _aligned(dn)
        with L.on_device_of(hidden):
            out = torch.empty(T, H, dtype=torch.bfloat16, device=dev)
            if T:
                ws = L.workspace(lib.b200moe_moe_fp8_block_ws_bytes(T, H, I, E, k), dev)
                L.check(lib.b200moe_moe_fp8_block_forward(hidden.data_ptr(), idx.data_ptr(), w.data_ptr(), gu.data_ptr(), gs.data_ptr(),
                                                          dn.data_ptr(), ds.data_ptr(), T, H, I, E, k, ws.data_ptr(), out.data_ptr(),
                                                          L.status_word(dev).data_ptr(), L.stream_of(hidden)))
        return out


def moe_fp8_block(hidden, top_k_indices, top_k_weights, gate_up_proj, gate_up_scale, down_proj, down_scale):
    """`moe` over 8-bit stacks, for serving: hidden (N,H) bf16, picks and weights (N,k), gate_up_proj (E,2I,H) and down_proj (E,H,I)
    float8_e4m3fn with scales (E, 2I/128, H/128) and (E, H/128, I/128) fp32 -> (N,H) bf16.  SiLU-GLU experts; H and I multiples of
    128; silu(gate) * up is requantised from fp32.  No backward: an input that requires a gradient is refused in grad mode (`moe` and
    `moe_mxfp8` train)."""
    fast = L.fast() if hidden.is_cuda else None
    if fast is not None:
        out = fast.moe_fp8_block(hidden, top_k_indices, top_k_weights, gate_up_proj, gate_up_scale, down_proj, down_scale,
                                 L.status_word(hidden.device))
        if out is not None:
            return out
    (hidden,) = (hidden.to(torch.get_autocast_dtype("cuda")),) if torch.is_autocast_enabled("cuda") else (hidden,)
    L.require_cuda_bf16("hidden", hidden)
    L.require(not (torch.is_grad_enabled() and (hidden.requires_grad or top_k_weights.requires_grad)),
              "moe_fp8_block has no backward: call it under torch.no_grad(), or train with moe or moe_mxfp8")
    dev, idx, w = hidden.device, top_k_indices, top_k_weights
    gu, gs = _weight("gate_up_proj", gate_up_proj, gate_up_scale, dev, 3)
    dn, ds = _weight("down_proj", down_proj, down_scale, dev, 3)
    L.require(hidden.dim() == 2, "hidden must be (N,H)")
    (T, H), (E, twoI, H2) = hidden.shape, gu.shape
    I = twoI // 2
    L.require(H2 == H and twoI % 2 == 0 and tuple(dn.shape) == (E, H, I), f"weight shapes must be (E,2I,H) and (E,H,I); got {tuple(gu.shape)}, "
              f"{tuple(dn.shape)}")
    L.require(H > 0 and I > 0 and H % BLOCK == 0 and I % BLOCK == 0, f"d_model and d_ff must be positive multiples of {BLOCK}, got {H}, {I}")
    L.require(idx.device == dev and idx.dtype == torch.int64 and idx.dim() == 2 and idx.shape[0] == T, "top_k_indices must be int64 (N,k)")
    L.require(w.device == dev and w.shape == idx.shape, "top_k_weights must be (N,k) on hidden's device")
    L.require(idx.shape[1] >= 1, "top_k_indices must have at least one pick a token")
    return _Experts.apply(hidden.contiguous(), idx.contiguous(), w.float().contiguous(), gu, gs, dn, ds)
