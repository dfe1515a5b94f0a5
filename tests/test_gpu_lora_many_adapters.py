"""GPU: as many adapters as a call may have, in stacks of more than 2^32 values.  Bounds as in tests/test_gpu_lora.py."""
import pytest
import torch

from .test_gpu_lora import BF, DEV, close, gen, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", ["K", "N"])
def test_65536_adapters(pkg, wide):
    L, R, T = 65536, 8, 700
    K, N = (16384, 64) if wide == "K" else (64, 16384)
    x, _, _, _, bs, _ = make(T, K, N, R, 1, seed=3)
    g = gen(4)
    a = torch.empty(L, R, K, dtype=BF, device=DEV).normal_(0.0, K ** -0.5, generator=g)
    b = torch.empty(L, N, R, dtype=BF, device=DEV).normal_(0.0, 0.3, generator=g)
    s = 0.5 + torch.rand(L, generator=g, device=DEV)
    index = torch.randint(0, L, (T,), generator=g, device=DEV)
    index[0], index[1], index[2], index[3:40] = L - 1, 0, -1, L - 2
    go = torch.randn(T, N, generator=g, device=DEV).to(BF)
    named = index.clamp(min=0).unique()
    ref = reference(x, a[named], b[named], s[named], bs, torch.where(index < 0, -1, torch.searchsorted(named, index)), go)
    for few in (True, False):
        rows = slice(0, 64) if few else slice(0, T)
        close(pkg.lora_linear(x[rows], a, b, index[rows], s, bs[rows]), tuple(t[rows] for t in ref["y"]), max(K, R))
    leaves = [t.requires_grad_() for t in (x, a, b)]
    gx, ga, gb = torch.autograd.grad(pkg.lora_linear(x, a, b, index, s, bs), leaves, go)
    close(gx, ref["gx"], max(N, R))
    close(ga[named], ref["ga"], max(N, T))
    close(gb[named], ref["gb"], max(K, T))
    none = torch.ones(L, dtype=torch.bool, device=DEV)
    none[named] = False
    for grad in (ga, gb):
        for part, of in zip(grad.split(4096), none.split(4096)):
            assert (part[of] == 0).all()
    pkg.check_status()
