"""GPU: `Fp8BlockMoELayer` picks the experts that the layer picks from which it was made, also where values are closer than fp32 resolves."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def near_ties(layer, H, E):
    """Hidden states (E/2,H) of which row i has the experts 2i and 2i+1 level to the last bit of their biases."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.zeros(E // 2, H, device=DEV)
    x[:, 0] = torch.linspace(0.5, 2.0, E // 2, device=DEV)
    x = x.to(torch.bfloat16)
    with torch.no_grad():
        layer.gate.weight.zero_()
        layer.gate.weight[:, 0] = torch.randn(E, generator=g, device=DEV)
        z = (x[:, :1].double() * layer.gate.weight[:, 0].double()).to(torch.bfloat16).double()
        s = torch.sigmoid(z)
        i = torch.arange(E // 2, device=DEV)
        layer.bias.zero_()
        layer.bias[1::2] = (s[i, 2 * i] - s[i, 2 * i + 1]).float()
    return x


@pytest.mark.parametrize("kw", [{}, dict(balance_loss=0.1), dict(z_loss=0.1), dict(scoring="softmax"), dict(num_groups=4, topk_groups=3)])
def test_same_picks(pkg, monkeypatch, kw):
    module, H, E, k = importlib.import_module(pkg.__name__ + ".layer"), 128, 64, 32
    torch.manual_seed(0)
    layer = pkg.MoELayer(H, 128, E, top_k=k, **kw).to(DEV).to(torch.bfloat16).eval()
    x = near_ties(layer, H, E)
    q = pkg.Fp8BlockMoELayer.from_layer(layer)
    if kw:
        want = pkg.fused_group_router(x, layer.gate.weight, layer.bias, k, E, layer.num_groups, layer.topk_groups, layer.scoring)[0]
    else:
        want = pkg.fused_mlp_router(x, layer.gate.weight, layer.bias, k, E)[0]
    seen, real = [], module.moe_fp8_block
    monkeypatch.setattr(module, "moe_fp8_block", lambda h, idx, *a: seen.append(idx) or real(h, idx, *a))
    q(x)
    assert torch.equal(seen[0], want) and q.exact_picks == bool(kw)
    if not kw:
        # the two routers differ here, so the choice between them shows
        other = pkg.Fp8BlockMoELayer(H, 128, E, k, device=DEV, exact_picks=True)
        other.load_state_dict(q.state_dict())
        other(x)
        assert not torch.equal(seen[1], want) and torch.equal(seen[1], pkg.fused_group_router(x, layer.gate.weight, layer.bias, k, E)[0])
    pkg.check_status()
