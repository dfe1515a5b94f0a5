"""GPU: weights and scales of the block-scaled products that require a gradient are refused in grad mode, compiled functions or not."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("compiled", [True, False])
def test_weights_that_require_a_gradient(pkg, monkeypatch, compiled):
    if not compiled:
        monkeypatch.setattr(importlib.import_module(pkg.__name__ + "._lib"), "fast", lambda: None)
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(20, 128, generator=g, device=DEV).to(torch.bfloat16)
    gu, gs = pkg.fp8_block_quantize_weight(torch.randn(4, 256, 128, generator=g, device=DEV).to(torch.bfloat16))
    dn, ds = pkg.fp8_block_quantize_weight(torch.randn(4, 128, 128, generator=g, device=DEV).to(torch.bfloat16))
    idx, wt = torch.arange(2, device=DEV).expand(20, 2), torch.ones(20, 2, device=DEV)
    param = torch.nn.Parameter

    def both(call, *tensors):
        want = call(*tensors)
        for i, t in enumerate(tensors):
            args = [*tensors]
            args[i] = param(t)
            with pytest.raises(ValueError, match="frozen.*requires_grad_"):
                call(*args)
            with torch.no_grad():
                assert torch.equal(call(*args), want)
            args[i] = param(t, requires_grad=False)
            assert torch.equal(call(*args), want)

    both(lambda w, s: pkg.fp8_block_linear(x, w, s), gu[0], gs[0])
    both(lambda w, s: pkg.fp8_block_linear(x.clone().requires_grad_(), w, s).detach(), gu[0], gs[0])
    both(lambda *t: pkg.moe_fp8_block(x, idx, wt, *t), gu, gs, dn, ds)
    pkg.check_status()
