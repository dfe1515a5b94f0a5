"""GPU: the compiled forms of the norm, of the products of codes and of the low-rank adapters against the Python Functions: the same bits and gradients,
and the Python Function for every call that is not plain."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16
NAMES = ("rms_norm", "fp8_block_linear_rows", "lora_linear", "fp8_block_linear")


@pytest.fixture()
def seen(pkg, monkeypatch):
    L = importlib.import_module(pkg.__name__ + "._lib")
    real = L.fast

    class Seen:
        taken, off = [], False

    s = Seen()
    s.taken = []
    for name in NAMES:
        def noting(*a, fn=getattr(real(), name), name=name):
            res = fn(*a)
            s.taken.append((name, res is not None))
            return res
        setattr(s, name, noting)
    monkeypatch.setattr(L, "fast", lambda: None if s.off or real() is None else s)
    return s


def tensors(T=90, K=256, N=136, R=16, n=3, shape=None):
    g = torch.Generator(device=DEV).manual_seed(T)
    r = lambda *sh: torch.randn(*sh, generator=g, device=DEV).to(BF)     # noqa: E731
    lead = shape or (T,)
    return dict(x=r(*lead, K), res=r(*lead, K), wn=1 + 0.1 * r(K), a=r(n, R, K) * 0.1, b=r(n, N, R), base=r(*lead, N),
                index=torch.randint(-1, n, lead, generator=g, device=DEV), s=torch.rand(n, generator=g, device=DEV), w=r(N, K))


def chain(pkg, t, grad, no_residual=False, no_base=False):
    """The three one after another: all outputs and gradients"""
    leaves = [t[k].detach().requires_grad_(grad) for k in ("x", "res", "wn", "a", "b", "base")]
    x, res, wn, a, b, base = leaves
    w, ws = pkg.fp8_block_quantize_weight(t["w"])
    out = pkg.rms_norm_fp8_block(x, wn, None if no_residual else res, return_norm=True)
    q, qs, y = out[:3]
    y2 = pkg.rms_norm(x, wn, None if no_residual else res)
    p = pkg.fp8_block_linear(y, w, ws, quantized=(q, qs))
    z = pkg.lora_linear(y, a, b, t["index"], t["s"], None if no_base else base)
    outs = [q.float(), qs, *out[2:], *([y2] if no_residual else y2), p, z]
    if not grad:
        with torch.no_grad():
            return outs + [pkg.fp8_block_linear(None, w, ws, quantized=(q, qs))]
    total = sum(o.float().square().sum() for o in outs[2:])
    return outs + list(torch.autograd.grad(total, leaves, allow_unused=True))


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("shape", [(90,), (300,), (4, 50), (2, 3, 64), (1,), ()])
@pytest.mark.parametrize("less", [False, True])
def test_same_bits(pkg, seen, grad, shape, less):
    t = tensors(shape=shape)
    here = chain(pkg, t, grad, less, less)
    assert seen.taken and all(ok for _, ok in seen.taken)
    count = len(seen.taken)
    seen.off = True
    there = chain(pkg, t, grad, less, less)
    assert len(seen.taken) == count and len(here) == len(there)
    for a, b in zip(here, there):
        assert (a is None) == (b is None)
        if a is not None:
            assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b) and a.requires_grad == b.requires_grad
    pkg.check_status()


def test_calls_that_are_not_plain(pkg, seen):
    """Strided rows, an index of another kind of memory, adapters in fp32, autocast, empty rows: the Python Function, with the same results."""
    t = tensors()
    w, ws = pkg.fp8_block_quantize_weight(t["w"])
    wide = torch.cat([t["x"], t["x"]], 1)[:, : t["x"].shape[1]]
    want = pkg.rms_norm(t["x"], t["wn"], t["res"])
    q, qs = pkg.rms_norm_fp8_block(t["x"], t["wn"])
    p = pkg.fp8_block_linear(None, w, ws, (q, qs))
    z = pkg.lora_linear(t["x"], t["a"], t["b"], t["index"], t["s"], t["base"])
    seen.taken.clear()
    assert all(torch.equal(a, b) for a, b in zip(pkg.rms_norm(wide, t["wn"], t["res"]), want))
    assert torch.equal(pkg.fp8_block_linear(None, w, ws, (q, qs.contiguous())), p)
    assert torch.equal(pkg.lora_linear(wide, t["a"], t["b"], t["index"], t["s"], t["base"]), z)
    assert torch.equal(pkg.lora_linear(t["x"], t["a"].float(), t["b"].float(), t["index"], t["s"], t["base"]), z)
    with torch.autocast("cuda", dtype=BF):
        assert torch.equal(pkg.lora_linear(t["x"], t["a"], t["b"], t["index"], t["s"], t["base"]), z)
        assert torch.equal(pkg.rms_norm(t["x"], t["wn"], t["res"])[0], want[0])
    assert pkg.lora_linear(t["x"][:0], t["a"], t["b"], t["index"][:0]).shape == (0, 136)
    assert seen.taken and not any(ok for _, ok in seen.taken)


@pytest.mark.parametrize("compiled", [True, False])
def test_second_derivatives_are_refused(pkg, seen, compiled):
    seen.off = not compiled
    t = tensors()
    for fn in (lambda x: pkg.rms_norm(x, t["wn"]), lambda x: pkg.lora_linear(x, t["a"], t["b"], t["index"])):
        x = t["x"].clone().requires_grad_()
        g, = torch.autograd.grad(fn(x).float().square().sum(), x, create_graph=True)
        assert torch.equal(g, torch.autograd.grad(fn(x).float().square().sum(), x)[0])
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.float().sum().backward()


@pytest.mark.parametrize("compiled", [True, False])
def test_a_changed_stream_is_noticed(pkg, seen, compiled):
    """h is both handed out and kept for the backward: in-place changes of it are an error there, as of any kept tensor."""
    seen.off = not compiled
    t = tensors()
    y, h = pkg.rms_norm(t["x"].clone().requires_grad_(), t["wn"], t["res"])
    with torch.no_grad():
        h.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.float().sum().backward()
