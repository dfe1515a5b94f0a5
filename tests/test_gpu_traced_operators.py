"""GPU: the routers' top-k and losses and the block-scaled products under a tracer and under forward-mode gradients.  A traced call gives on other
inputs, of another size too, what the plain call gives; an input with a tangent is refused."""
import importlib

import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning"), pytest.mark.filterwarnings("ignore::DeprecationWarning")]
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def stacks(pkg, E=8, H=256, I=128):
    g = gen(1)
    gu = (torch.randn(E, 2 * I, H, generator=g, device=DEV) * 0.1).to(torch.bfloat16)
    dn = (torch.randn(E, H, I, generator=g, device=DEV) * 0.1).to(torch.bfloat16)
    return (*pkg.fp8_block_quantize_weight(gu), *pkg.fp8_block_quantize_weight(dn))


def calls(pkg):
    """name -> (function of floating-point tensors, the tensors of a batch n)"""
    gu, gs, dn, ds = stacks(pkg)
    w, s = gu[0], gs[0]
    bias = torch.randn(64, generator=gen(2), device=DEV) * 0.1

    def logits(n):
        return (torch.randn(n, 30, 64, generator=gen(n), device=DEV),)

    def hidden(n, *shape):
        return (torch.randn(*shape, n, 256, generator=gen(n), device=DEV).to(torch.bfloat16),)

    def picked(n):
        return (*hidden(n), torch.rand(n, 3, generator=gen(n), device=DEV))

    def losses(z, per_sequence):
        return pkg.router_losses(z, torch.topk(z, 3, dim=-1).indices, "softmax", None, per_sequence)

    return {
        "topk": (lambda z: pkg.group_topk(z, 6, bias, 8, 3, return_counts=True), logits),
        "topk, no bias": (lambda z: pkg.group_topk(z, 6, scoring="softmax"), logits),
        "losses": (lambda z: losses(z, False), logits),
        "losses by sequence": (lambda z: losses(z, True), logits),
        "linear": (lambda x: pkg.fp8_block_linear(x, w, s), lambda n: hidden(n, 2)),
        "quantiser": (lambda x: [t.float() for t in pkg.fp8_block_quantize(x)], hidden),
        "weights' quantiser": (lambda x: [t.float() for t in pkg.fp8_block_quantize_weight(x)], hidden),
        "experts": (lambda x, wt: pkg.moe_fp8_block(x, torch.arange(3, device=DEV).expand(x.shape[0], 3), wt, gu, gs, dn, ds), picked),
    }


NAMES = ["topk", "topk, no bias", "losses", "losses by sequence", "linear", "quantiser", "weights' quantiser", "experts"]


def flat(out):
    return out if isinstance(out, (tuple, list)) else (out,)


@pytest.mark.parametrize("name", NAMES)
def test_traced(pkg, name):
    fn, inputs = calls(pkg)[name]
    with torch.no_grad():
        traced = torch.jit.trace(fn, inputs(40))
        for n in (40, 7, 300):
            args = tuple(t + 0.5 for t in inputs(n))
            junk = [torch.full((1 << 16,), 0x5a, dtype=torch.uint8, device=DEV) for _ in range(4)]      # what unwritten memory would hold
            del junk
            for a, b in zip(flat(traced(*args)), flat(fn(*args))):
                assert a.dtype == b.dtype and torch.equal(a, b), n
    pkg.check_status()


@pytest.mark.parametrize("kw", [{}, dict(num_groups=4, topk_groups=2), dict(scoring="softmax", balance_loss=0.1)])
@pytest.mark.parametrize("eight", [False, True])
def test_traced_layer(pkg, kw, eight):
    torch.manual_seed(0)
    layer = pkg.MoELayer(256, 128, 16, top_k=3, **kw).to(DEV).to(torch.bfloat16).eval()
    if eight:
        layer = pkg.Fp8BlockMoELayer.from_layer(layer)
    x = [torch.randn(n, 20, 256, generator=gen(n), device=DEV).to(torch.bfloat16) for n in (2, 5)]
    with torch.no_grad():
        layer(x[0])          # a layer reads its act codes in its first call
        traced = torch.jit.trace(layer, (x[0],))
        for t in x:
            assert torch.equal(traced(t), layer(t))
    pkg.check_status()


@pytest.mark.parametrize("name", NAMES)
def test_forward_gradients_are_refused(pkg, name):
    """As `moe` refuses them, whichever input has the tangent."""
    fn, inputs = calls(pkg)[name]
    args = inputs(20)
    gu, gs, dn, ds = stacks(pkg)
    codes = torch.zeros(8, dtype=torch.int32, device=DEV)
    with fw.dual_level():
        x = fw.make_dual(torch.zeros(20, 256, dtype=torch.bfloat16, device=DEV), torch.ones(20, 256, dtype=torch.bfloat16, device=DEV))
        with pytest.raises(Exception) as moe:
            pkg.moe(x, torch.zeros(20, 1, dtype=torch.int64, device=DEV), torch.ones(20, 1, device=DEV), gu.to(torch.bfloat16), dn.to(torch.bfloat16),
                    codes)
        for i, t in enumerate(args):
            dual = [*args]
            dual[i] = fw.make_dual(t, torch.ones_like(t))
            with pytest.raises(moe.type):
                fn(*dual)
        if name == "linear":
            with pytest.raises(moe.type):
                pkg.fp8_block_linear(args[0], gu[0], fw.make_dual(gs[0], torch.ones_like(gs[0])))
    fn(*args)
    pkg.check_status()


def test_quantisers_of_parameters(pkg):
    """A tensor that requires a gradient is quantised; its codes and scales do not require one."""
    p = torch.nn.Parameter(torch.randn(200, 256, generator=gen(0), device=DEV).to(torch.bfloat16))
    for fn in (pkg.fp8_block_quantize, pkg.fp8_block_quantize_weight):
        for a, b in zip(fn(p), fn(p.detach())):
            assert not a.requires_grad and torch.equal(a.float(), b.float())


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_inference_mode(pkg, monkeypatch, name, compiled):
    """Results, and inputs made in inference mode and used outside it."""
    if not compiled:
        monkeypatch.setattr(importlib.import_module(pkg.__name__ + "._lib"), "fast", lambda: None)
    fn, inputs = calls(pkg)[name]
    want = flat(fn(*inputs(20)))
    with torch.inference_mode():
        args = inputs(20)
        here = flat(fn(*args))
    for got in (here, flat(fn(*args))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    pkg.check_status()
