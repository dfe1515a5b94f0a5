"""GPU: gradients of the norm for rows in other places and orders, and for a residual that rows share.  Bounds as in tests/test_gpu_norm.py."""
import pytest
import torch

from .test_gpu_norm import BF, DEV, EPS, F32, HF, close, gen, make, norm64

pytestmark = pytest.mark.gpu


def gradients64(h, w, gy, gh):
    """(of h, its size, of w, its size)"""
    n, rstd = norm64(h, torch.ones_like(w))
    d = gy.double() * w.double()
    back = (d * n).mean(-1, keepdim=True)
    gw = (gy.double() * n).reshape(-1, h.shape[-1])
    return (rstd * (d - n * back) + gh.double(), rstd * (d.abs() + n.abs() * (d * n).abs().mean(-1, keepdim=True)) + gh.double().abs(),
            gw.sum(0), gw.abs().sum(0))


@pytest.mark.parametrize("K", [1040, 136, 37])
def test_layouts(pkg, K):
    T = 40
    wide = torch.randn(T, 3 * K + 5, generator=gen(0), device=DEV).to(BF)
    _, r, w = make(T, K, BF)
    views = [lambda t: t[:, :K], lambda t: t[:, K:2 * K], lambda t: t[:, 3:3 + K], lambda t: t[::2, 1:1 + K], lambda t: t[:, : 2 * K : 2], lambda t: t[3, :K],
             lambda t: t[:, :K].unflatten(0, (5, 8)), lambda t: t[:, :K].unflatten(0, (5, 8)).transpose(0, 1), lambda t: t[:, :K].t().contiguous().t()]
    for view in views:
        leaf, w1 = wide.clone().requires_grad_(), w.clone().requires_grad_()
        x = view(leaf)
        r1 = r[: x.numel() // K].reshape(x.shape).clone().requires_grad_()
        gy, gh = (torch.randn(x.shape, generator=gen(i), device=DEV).to(BF) for i in (1, 2))
        y, h = pkg.rms_norm(x, w1, r1, EPS)
        gx, gr, gw = torch.autograd.grad([y, h], [leaf, r1, w1], [gy, gh])
        ref, size, refw, sizew = gradients64(h.detach(), w, gy, gh)
        close(gr, ref, size, 2.0 ** -17)
        close(gw, refw, sizew, 2.0 ** -17)
        other = wide.clone().requires_grad_()
        assert torch.equal(gx, torch.autograd.grad(view(other), other, gr)[0])
        # without a residual, and with gradients that are views themselves
        y = pkg.rms_norm(x, w1, eps=EPS)
        gx, gw = torch.autograd.grad(y, [x, w1], torch.cat([gy, gy], -1)[..., :K])
        ref, size, refw, sizew = gradients64(x.detach(), w, gy, torch.zeros_like(gy))
        close(gx, ref, size, 2.0 ** -17)
        close(gw, refw, sizew, 2.0 ** -17)


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("T,K", [(40, 1040), (40, 37), (3000, 136)])
def test_a_residual_that_rows_share(pkg, dt, T, K):
    """Its gradient is the sum over the rows: each row's is off by half a step of its type and by 2^-17 of its size, and the sum, in fp32 or better, is rounded once more."""
    x, r, w = make(T, K, dt, seed=3)
    one = r[0].clone().requires_grad_()
    leaf, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
    gy, gh = (torch.randn(T, K, generator=gen(i), device=DEV).to(dt) for i in (1, 2))
    y, h = pkg.rms_norm(leaf, w1, one.expand(T, K), EPS)
    gx, g1, gw = torch.autograd.grad([y, h], [leaf, one, w1], [gy, gh])
    ref, size, refw, sizew = gradients64(h.detach(), w, gy, gh)
    close(gx, ref, size, 2.0 ** -17)
    close(gw, refw, sizew, 2.0 ** -17)
    half, terms = torch.finfo(dt).eps / 2, T * 2.0 ** -24
    lim = half * ref.sum(0).abs() * (1 + 2.0 ** -6) + (1 + half) * ((half * (1 + 2.0 ** -17) + terms) * ref.abs() + 2.0 ** -17 * size).sum(0) + 2.0 ** -24
    assert g1.dtype == dt and ((g1.double() - ref.sum(0)).abs() <= lim).all()
    # the rows' gradients as they came out, summed
    assert ((g1.double() - gx.double().sum(0)).abs() <= half * gx.double().sum(0).abs() * (1 + 2.0 ** -6) + 2 * terms * gx.double().abs().sum(0) + 2.0 ** -24).all()
