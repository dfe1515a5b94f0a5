"""GPU: `router_losses` against a 64-bit restatement.

Steps of 2^-23 (fp32): a probability is off by at most 2 (exponential) + 2 (those of the sum) + 6.5 (additions) + 2, sigmoid scores by
twice that; its sums over a warp's tokens (2048 at most here) by 2048 / 2 in the worst case, in practice by the square root of it: the worst
case is what is allowed, 2^-12 relative for P, of positive terms.  lse is off by 2^-20 (1 + |lse|), its square by twice that.  A gradient is a
difference of terms p f and p <f, p>, with 2^-17 of their size (f comes from whole numbers), plus its rounding."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def losses64(z, idx, scoring, mask, per_sequence, gb, gz):
    """balance, z, grad and the size of the gradient's terms; z (B,S,E)"""
    z = z.double()
    B, S, E = z.shape
    m = (torch.ones(B, S, dtype=torch.bool, device=z.device) if mask is None else mask.clone()) & ~(z == -torch.inf).all(2)
    soft = torch.softmax(z, 2)
    p = soft if scoring == "softmax" else torch.softmax(torch.nn.functional.logsigmoid(z), 2)
    lse = torch.logsumexp(z, 2)
    N = m.sum()
    grad, size = torch.zeros_like(z), torch.zeros_like(z)
    zl = torch.where(m, lse ** 2, 0.0 * lse.nan_to_num(0, 0, 0)).sum() / N.clamp(min=1)
    parts = [slice(b, b + 1) for b in range(B)] if per_sequence else [slice(0, B)]
    live = sum(int(m[b].any()) for b in parts)
    balance = torch.zeros((), dtype=torch.float64, device=z.device)
    for b in parts:
        n = m[b].sum()
        if n == 0:
            continue
        f = torch.bincount(idx[b][m[b]].reshape(-1), minlength=E).double() * E / (idx.shape[2] * n)
        balance += (f * p[b][m[b]].mean(0)).sum() / live
        dot = (p[b] * f).sum(2, keepdim=True)
        one = torch.sigmoid(-z[b]) if scoring == "sigmoid" else torch.ones_like(z[b])
        grad[b] = gb * p[b] * (f - dot) * one / (n * live)
        size[b] = abs(gb) * p[b] * (f + dot) * one / (n * live)
    gl = gz * 2 * (lse / N.clamp(min=1))[..., None] * soft
    grad = torch.where(m[..., None], grad + gl, torch.zeros_like(grad))
    size = torch.where(m[..., None], size + gl.abs() + abs(gz) * 2.0 / N.clamp(min=1) * soft, torch.zeros_like(grad))
    return balance, zl, grad, size


def make(B, S, E, k, dtype, seed, masked):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = (torch.randn(B, S, E, generator=g, device=DEV) * 1.5).to(dtype)
    idx = torch.topk(z.float() + torch.randn(B, S, E, generator=g, device=DEV), k, dim=-1).indices
    mask = None
    if masked:
        mask = torch.arange(S, device=DEV)[None] < torch.randint(0, S + 1, (B, 1), generator=g, device=DEV)
        mask[-1] = True
    return z, idx, mask


SHAPES = [(1, 1, 1, 1), (1, 1, 256, 8), (1, 63, 8, 2), (2, 65, 60, 4), (1, 512, 8, 2), (5, 129, 96, 6), (16, 333, 64, 6), (3, 7000, 33, 3), (1, 30000, 256, 8),
          (300, 3, 128, 2), (1, 30000, 2, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,masked,per_sequence", list(itertools.product(("softmax", "sigmoid"), (False, True), (False, True))))
def test_losses_and_gradient(pkg, dtype, scoring, masked, per_sequence):
    gb, gz = torch.tensor(0.7, device=DEV), torch.tensor(0.02, device=DEV)
    for n, (B, S, E, k) in enumerate(SHAPES):
        z, idx, mask = make(B, S, E, k, dtype, n, masked)
        z.requires_grad_(True)
        got = pkg.router_losses(z, idx, scoring, mask, per_sequence)
        (grad,) = torch.autograd.grad(got, z, (gb, gz))
        b, zl, rg, size = losses64(z.detach(), idx, scoring, mask, per_sequence, 0.7, 0.02)
        assert abs(float(got[0].detach()) - float(b)) <= 2.0 ** -12 * float(b), (B, S, E, float(got[0]), float(b))
        assert abs(float(got[1].detach()) - float(zl)) <= 2.0 ** -18 * (1 + float(zl)), (B, S, E)
        bound = 2.0 ** -17 * size + torch.finfo(dtype).eps / 2 * rg.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert grad.dtype == dtype and ((grad.double() - rg).abs() <= bound).all(), (B, S, E, float(((grad.double() - rg).abs() / bound).max()))
        again = pkg.router_losses(z.detach(), idx, scoring, mask, per_sequence)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])       # the same bits, also without a gradient


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_gradient_is_what_differences_give(pkg, scoring):
    """Central differences, h = 2^-5, along a unit direction over 8 tokens of 16 experts: truncation h^2 / 6 times a third derivative below 8 for
    the balance and below 40 for z (lse < 6): 7e-3 at most; the losses' own 2^-18 (1 + z) over 2h: 2e-3."""
    g = torch.Generator(device=DEV).manual_seed(0)
    z = torch.randn(8, 16, generator=g, device=DEV).requires_grad_(True)
    idx = torch.topk(z.detach(), 3, dim=1).indices
    d = torch.nn.functional.normalize(torch.randn(8, 16, generator=g, device=DEV).flatten(), dim=0).view(8, 16)
    h = 2.0 ** -5
    for i in range(2):
        (dz,) = torch.autograd.grad(pkg.router_losses(z, idx, scoring)[i], z)
        up, dn = (pkg.router_losses((z + s * h * d).detach(), idx, scoring)[i] for s in (1, -1))
        num = (float(up) - float(dn)) / (2 * h)
        assert abs(float((dz * d).sum()) - num) <= 9e-3 * (1 if i else 0.2), (scoring, i)


def test_tokens_that_do_not_count(pkg):
    """Masked tokens may hold anything; a token of -inf counts never; no tokens at all give zeros."""
    z, idx, _ = make(2, 200, 64, 6, torch.float32, 1, False)
    mask = torch.rand(2, 200, generator=torch.Generator().manual_seed(0)).to(DEV) < 0.5
    for scoring, seq in itertools.product(("softmax", "sigmoid"), (False, True)):
        a = z.clone().requires_grad_(True)
        ref = pkg.router_losses(a, idx, scoring, mask, seq)
        ga = torch.autograd.grad(ref[0] + ref[1], a)[0]
        dirty = z.clone()
        dirty[~mask] = torch.nan
        dirty.requires_grad_(True)
        bad = idx.clone()
        bad[~mask] = -7
        got = pkg.router_losses(dirty, bad, scoring, mask.to(torch.int32), seq)
        gd = torch.autograd.grad(got[0] + got[1], dirty)[0]
        assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1]) and torch.equal(ga, gd) and (gd[~mask] == 0).all()
        low = z.clone()
        low[~mask] = -torch.inf
        low.requires_grad_(True)
        got = pkg.router_losses(low, idx, scoring, None, seq)
        gl = torch.autograd.grad(got[0] + got[1], low)[0]
        assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1]) and torch.equal(ga, gl)
        none = z.clone().requires_grad_(True)
        got = pkg.router_losses(none, idx, scoring, torch.zeros_like(mask), seq)
        assert float(got[0]) == 0 and float(got[1]) == 0 and (torch.autograd.grad(got[0] + got[1], none)[0] == 0).all()
    pkg.check_status()
    empty = torch.empty(0, 64, device=DEV, requires_grad=True)
    got = pkg.router_losses(empty, torch.empty(0, 6, dtype=torch.int64, device=DEV))
    assert float(got[0]) == 0 and torch.autograd.grad(got[0] + got[1], empty)[0].shape == (0, 64)


def test_far_logits_and_picks_out_of_range(pkg):
    z = torch.full((300, 32), -300.0, device=DEV)      # every sigmoid is 0 in fp32
    z[:, 3] = -299.0
    z[7] = 90.0
    z[8, 5] = -torch.inf
    z.requires_grad_(True)
    idx = torch.zeros(300, 2, dtype=torch.int64, device=DEV)
    idx[:, 1] = 3
    for scoring in ("softmax", "sigmoid"):
        got = pkg.router_losses(z, idx, scoring)
        b, zl, rg, size = losses64(z.detach()[None], idx[None], scoring, None, False, 1.0, 1.0)
        (g,) = torch.autograd.grad(got[0] + got[1], z)
        assert abs(float(got[0].detach()) - float(b)) <= 2.0 ** -12 * float(b) and abs(float(got[1].detach()) - float(zl)) <= 2.0 ** -18 * (1 + float(zl))
        # exponents of 300 carry 300 * 2^-24 of their own
        assert ((g.double() - rg[0]).abs() <= 2.0 ** -14 * size[0] + 1e-12).all()
    pkg.check_status()
    idx[5, 0], idx[6, 1] = 32, -1
    got = pkg.router_losses(z.detach(), idx)
    with pytest.raises(RuntimeError, match="expert index"):
        pkg.check_status()
    assert torch.isfinite(got[0])
    for none in (idx[:, :0], idx.repeat(1, 2)[:, ::2][:, :0]):
        with pytest.raises(ValueError):
            pkg.router_losses(z.detach(), none)


def test_strides_other_stream_and_captured_graph(pkg):
    z, idx, mask = make(4, 500, 64, 6, torch.bfloat16, 2, True)
    ref = pkg.router_losses(z, idx, "softmax", mask, True)
    wide = torch.empty(4, 500, 80, dtype=torch.bfloat16, device=DEV)
    wide[..., 5:69] = z
    a = pkg.router_losses(wide[..., 5:69], idx.transpose(0, 1).contiguous().transpose(0, 1), "softmax", mask.t().contiguous().t(), True)
    assert torch.equal(a[0], ref[0]) and torch.equal(a[1], ref[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = torch.zeros_like(z).requires_grad_(True)
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(sum(pkg.router_losses(static, idx, "softmax", mask, True)), static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.router_losses(static, idx, "softmax", mask, True)
        (grad,) = torch.autograd.grad(out[0] + out[1], static)
    with torch.no_grad():
        static.copy_(z)
    for _ in range(2):
        graph.replay()
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    z.requires_grad_(True)
    assert torch.equal(grad, torch.autograd.grad(sum(pkg.router_losses(z, idx, "softmax", mask, True)), z)[0])
