"""GPU: the compiled forms of the routers' top-k and losses and of the block-scaled products against the Python Functions: the same bits and
gradients, and the Python Function for every call that is not plain."""
import importlib

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("group_topk", "router_losses", "fp8_block_linear", "moe_fp8_block")


class Seen:
    def __init__(self, module):
        self.taken = []
        for name in NAMES:
            setattr(self, name, self._noting(getattr(module, name)))

    def _noting(self, fn):
        def call(*a):
            res = fn(*a)
            self.taken.append(res is not None)
            return res
        return call


@pytest.fixture()
def seen(pkg, monkeypatch):
    L = importlib.import_module(pkg.__name__ + "._lib")
    real = L.fast
    s = Seen(real())
    s.off = False
    monkeypatch.setattr(L, "fast", lambda: None if s.off or real() is None else s)
    return s


def call(pkg, kind, grad=True, **change):
    """(outputs, gradients)"""
    g = torch.Generator(device=DEV).manual_seed(3)
    z = (change.get("z") if "z" in change else torch.randn(4, 90, 64, generator=g, device=DEV).to(torch.bfloat16)).detach().requires_grad_(grad)
    if kind == "topk":
        b = change.get("b", torch.randn(64, generator=g, device=DEV) * 0.1)
        idx, w, c = pkg.group_topk(z, 6, b, 8, 3, return_counts=True)
        return (idx, w, c), torch.autograd.grad(w, z, torch.ones_like(w)) if grad else ()
    if kind == "losses":
        idx = torch.topk(z.detach().float(), 6, dim=-1).indices
        mask = change.get("mask", torch.rand(z.shape[:-1], generator=g, device=DEV) < 0.8)
        r = pkg.router_losses(z, idx, "sigmoid", mask, True)
        return r, torch.autograd.grad(r[0] + 0.5 * r[1], z) if grad else ()
    w = (torch.randn(8, 256, 128, generator=g, device=DEV) * 20).to(torch.float8_e4m3fn)
    s = torch.rand(8, 2, 1, generator=g, device=DEV) * 1e-3
    if kind == "linear":
        x = change.get("x", torch.randn(3, 40, 128, generator=g, device=DEV).to(torch.bfloat16)).detach().requires_grad_(grad)
        y = pkg.fp8_block_linear(x, w[0], s[0])
        return (y,), torch.autograd.grad(y, x, torch.ones_like(y)) if grad else ()
    x = change.get("x", torch.randn(120, 128, generator=g, device=DEV).to(torch.bfloat16))
    d, ds = w.view(8, 128, 256), s.view(8, 1, 2)
    idx = torch.topk(torch.randn(120, 8, generator=g, device=DEV), 2, dim=1).indices
    wt = change.get("wt", torch.rand(120, 2, generator=g, device=DEV))
    return (pkg.moe_fp8_block(x, idx, wt, w, s, d[:, :, :128].contiguous(), ds[..., :1].contiguous()),), ()


@pytest.mark.parametrize("kind", ["topk", "losses", "linear", "experts"])
@pytest.mark.parametrize("grad", [True, False])
def test_same_bits(pkg, seen, kind, grad):
    here = call(pkg, kind, grad)
    assert seen.taken and all(seen.taken)
    n = len(seen.taken)
    seen.off = True
    there = call(pkg, kind, grad)
    assert len(seen.taken) == n
    for a, b in zip(here[0] + tuple(here[1]), there[0] + tuple(there[1])):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)
        assert a.requires_grad == b.requires_grad


@pytest.mark.parametrize("compiled", [True, False])
def test_a_second_derivative_is_refused(pkg, seen, compiled):
    """The gradients are right under create_graph, and going through them is an error, not a zero."""
    seen.off = not compiled
    z = torch.randn(20, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0), requires_grad=True)
    x = torch.randn(20, 128, device=DEV).to(torch.bfloat16).requires_grad_(True)
    w, s = torch.ones(64, 128, device=DEV).to(torch.float8_e4m3fn), torch.ones(1, 1, device=DEV)
    idx, weights = pkg.group_topk(z, 4)
    for out, leaf in ((weights.square().sum(), z), (sum(pkg.router_losses(z, idx)), z), (pkg.fp8_block_linear(x, w, s).float().square().sum(), x)):
        (plain,) = torch.autograd.grad(out, leaf, retain_graph=True)
        (g,) = torch.autograd.grad(out, leaf, create_graph=True)
        assert torch.equal(plain, g)
        with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
            g.float().sum().backward()


class Noting(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_other_calls_go_to_the_python_functions(pkg, seen):
    g = torch.Generator(device=DEV).manual_seed(3)
    z = torch.randn(4, 90, 64, generator=g, device=DEV).to(torch.bfloat16)
    want = call(pkg, "topk", z=z)
    seen.taken.clear()
    wide = torch.zeros(4, 90, 80, dtype=torch.bfloat16, device=DEV)
    wide[..., :64] = z
    b = torch.randn(64, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    for got in (call(pkg, "topk", z=wide[..., :64]),):
        assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[1][0], want[1][0])
    call(pkg, "topk", b=b.double())
    call(pkg, "losses", mask=torch.ones(4, 90, device=DEV))
    call(pkg, "linear", x=torch.zeros(3, 128, 40, dtype=torch.bfloat16, device=DEV).transpose(1, 2))
    call(pkg, "experts", wt=torch.rand(120, 2, dtype=torch.float64, device=DEV))
    with Noting():
        call(pkg, "experts")
        call(pkg, "linear")
    assert not any(seen.taken)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = pkg.fp8_block_linear(torch.zeros(5, 128, device=DEV), torch.zeros(64, 128, device=DEV).to(torch.float8_e4m3fn), torch.ones(1, 1, device=DEV))
    assert out.dtype == torch.bfloat16 and not any(seen.taken)


def test_refusals_on_the_gpu(pkg):
    z = torch.zeros(4, 64, device=DEV)
    w8, s8 = torch.zeros(64, 128, device=DEV).to(torch.float8_e4m3fn), torch.ones(1, 1, device=DEV)
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device=DEV)
    idx, wt = torch.zeros(4, 2, dtype=torch.int64, device=DEV), torch.zeros(4, 2, device=DEV)
    gu, gs = torch.zeros(4, 256, 128, device=DEV).to(torch.float8_e4m3fn), torch.ones(4, 2, 1, device=DEV)
    dn, ds = torch.zeros(4, 128, 128, device=DEV).to(torch.float8_e4m3fn), torch.ones(4, 1, 1, device=DEV)
    for text, call in [
            ("top_k", lambda: pkg.group_topk(z, 0)), ("top_k = 9", lambda: pkg.group_topk(z, 9, None, 8, 1)), ("groups", lambda: pkg.group_topk(z, 4, None, 7)),
            ("open groups", lambda: pkg.group_topk(z, 4, None, 8, 9)), ("float32, got", lambda: pkg.group_topk(z.double(), 4)),
            ("E elements", lambda: pkg.group_topk(z, 4, torch.zeros(3, device=DEV))), ("E = 257", lambda: pkg.group_topk(torch.zeros(4, 257, device=DEV), 4)),
            ("top_k_indices", lambda: pkg.router_losses(z, idx.int())), ("top_k_indices", lambda: pkg.router_losses(z, idx[:3])),
            ("per_sequence", lambda: pkg.router_losses(z, idx, per_sequence=True)), ("mask", lambda: pkg.router_losses(z, idx, mask=torch.ones(3, device=DEV))),
            ("got torch.float64", lambda: pkg.router_losses(z.double(), idx)),
            ("bfloat16", lambda: pkg.fp8_block_linear(x.float(), w8, s8)), ("float8_e4m3fn", lambda: pkg.fp8_block_linear(x, x, s8)),
            ("scale of weight", lambda: pkg.fp8_block_linear(x, w8, s8.double())), ("scale of weight", lambda: pkg.fp8_block_linear(x, w8, torch.ones(1, 2, device=DEV))),
            ("x must be", lambda: pkg.fp8_block_linear(x[:, :64], w8, s8)), ("multiple of 8", lambda: pkg.fp8_block_linear(x, w8[:12], s8)),
            ("multiple of 8", lambda: pkg.fp8_block_linear(x[:, :24], w8[:, :24], s8)), ("on the input's device", lambda: pkg.fp8_block_linear(x, w8.cpu(), s8)),
            ("multiple of 8", lambda: pkg.fp8_block_quantize(x[:, :12])), ("no backward", lambda: pkg.moe_fp8_block(x.requires_grad_(), idx, wt, gu, gs, dn, ds)),
            ("no backward", lambda: pkg.moe_fp8_block(x.detach(), idx, wt.clone().requires_grad_(), gu, gs, dn, ds)),
            ("multiples of 128", lambda: pkg.moe_fp8_block(x.detach()[:, :64], idx, wt, gu[..., :64].contiguous(), gs, dn[:, :64].contiguous(), ds)),
            ("weight shapes", lambda: pkg.moe_fp8_block(x.detach(), idx, wt, gu, gs, dn[:3], ds[:3])),
            ("top_k_indices", lambda: pkg.moe_fp8_block(x.detach(), idx[:3], wt, gu, gs, dn, ds)),
            ("top_k_weights", lambda: pkg.moe_fp8_block(x.detach(), idx, wt[:, :1], gu, gs, dn, ds))]:
        with pytest.raises(ValueError, match=text):
            call()
    pkg.check_status()
