"""GPU: gradients of the adapters where the CTAs of the factors' gradient are no multiple of the clusters of the launch that they share with u = g B.  Bounds as in
tests/test_gpu_lora.py."""
import pytest
import torch

from .test_gpu_lora import BF, DEV, F32, close, gen, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,K,N,R,n,how", [(1000, 136, 2176, 16, 3, "packed"), (1000, 136, 2176, 64, 1, "one"), (200, 264, 648, 24, 5, "mixed"), (600, 64, 1032, 128, 33, "mixed"),
                                           (1000, 136, 2176, 32, 101, "mixed")])
def test_gradients(pkg, T, K, N, R, n, how, dtype):
    x, a, b, s, bs, index = make(T, K, N, R, n, how, seed=31, dtype=dtype)
    go = torch.randn(T, N, generator=gen(32), device=DEV).to(BF)
    leaves = [t.requires_grad_() for t in (x, a, b)]
    grads = torch.autograd.grad(pkg.lora_linear(x, a, b, index, s, bs), leaves, go)
    ref = reference(x.detach(), a.detach(), b.detach(), s, bs, index, go)
    for got, name, terms in zip(grads, ("gx", "ga", "gb"), (max(N, R), max(N, T), max(K, T))):
        close(got, ref[name], terms)
    for i, want in enumerate(grads):       # each by itself
        args = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, a, b))]
        assert torch.equal(torch.autograd.grad(pkg.lora_linear(*args, index, s, bs), args[i], go)[0], want)
    pkg.check_status()
