"""GPU: the observer is told of the group top-k, the router losses and the block-scaled products, by whichever path they are reached, with the
launches they make."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("compiled", [True, False])
def test_observer_is_told(pkg, monkeypatch, compiled):
    if not compiled:
        monkeypatch.setattr(importlib.import_module(pkg.__name__ + "._lib"), "fast", lambda: None)
    g = torch.Generator(device=DEV).manual_seed(0)
    z = torch.randn(4, 100, 64, generator=g, device=DEV).requires_grad_()
    idx = torch.topk(z.detach(), 4, dim=-1).indices
    x = torch.randn(300, 256, generator=g, device=DEV).to(torch.bfloat16).requires_grad_()
    gu, gs = pkg.fp8_block_quantize_weight(torch.randn(8, 512, 256, generator=g, device=DEV).to(torch.bfloat16))
    dn, ds = pkg.fp8_block_quantize_weight(torch.randn(8, 256, 256, generator=g, device=DEV).to(torch.bfloat16))
    picks, wt = torch.arange(2, device=DEV).expand(300, 2), torch.ones(300, 2, device=DEV)
    torch.cuda.synchronize()

    def seen(call):
        names = []
        pkg.ops.set_hook(lambda name, launches, a, b: names.append((name, launches)))
        try:
            call()
        finally:
            pkg.ops.set_hook(None)
        torch.cuda.synchronize()
        return names

    assert seen(lambda: pkg.group_topk(z, 4)[1].sum().backward()) == [("group_topk_fwd", 1), ("group_topk_bwd", 1)]
    for rows, per_sequence, launches in ((z[:1, :8], False, 1), (z, False, 2), (z, True, 3)):
        picked = idx[: rows.shape[0], : rows.shape[1]].contiguous()
        got = seen(lambda: sum(pkg.router_losses(rows.contiguous(), picked, "softmax", None, per_sequence)).backward())
        assert got == [("router_losses_fwd", launches), ("router_losses_bwd", 1)]
    # 300 rows both ways; 4 rows are quantised by the product
    assert seen(lambda: pkg.fp8_block_linear(x, gu[0], gs[0]).sum().backward()) == [("fp8_block_quant", 1), ("fp8_block_linear", 1)] * 2
    assert seen(lambda: pkg.fp8_block_linear(x.detach()[:4], gu[0], gs[0])) == [("fp8_block_linear", 1)]
    assert seen(lambda: pkg.fp8_block_quantize(x)) == [("fp8_block_quant", 1)]
    assert seen(lambda: pkg.fp8_block_quantize_weight(x)) == [("fp8_block_quant_weight", 1)]
    got = [n for n, _ in seen(lambda: pkg.moe_fp8_block(x.detach(), picks, wt, gu, gs, dn, ds))]
    assert got == ["permute_build", "fp8_block_quant", "fp8_block_gate_up", "fp8_block_down", "combine"]
    pkg.check_status()
