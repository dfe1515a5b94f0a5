"""CPU and GPU: layers out of pickles and copies."""
import copy
import io

import pytest
import torch

from tests.conftest import load_pkg

ADDED = ("scoring", "num_groups", "topk_groups", "group_score", "balance_loss", "z_loss", "balance_per_sequence", "aux_loss")


def before(layer):
    """The layer as a pickle holds it that was written before it had groups of experts and losses."""
    old = copy.deepcopy(layer)
    for name in ADDED:
        del old.__dict__[name]
    buf = io.BytesIO()
    torch.save(old, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


def test_a_layer_without_the_routers_attributes():
    layer = load_pkg().MoELayer(64, 72, 8, top_k=2)
    old = before(layer)
    assert not set(ADDED) & set(old.__dict__) - {"aux_loss"} and old._plain_router() and old.aux_loss is None
    assert [getattr(old, n) for n in ADDED] == [getattr(layer, n) for n in ADDED]


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["bf16", "mxfp8"])
def test_it_runs_as_it_did(pkg, precision):
    torch.manual_seed(0)
    layer = pkg.MoELayer(128, 128, 8, top_k=2, precision=precision).to("cuda").to(torch.bfloat16)
    old = before(layer)
    x = torch.randn(3, 20, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(torch.bfloat16)
    for mod in (layer, old):
        mod.zero_grad()
        mod(x).float().square().mean().backward()
    assert torch.equal(old(x), layer(x)) and old.aux_loss is None
    for a, b in zip(old.parameters(), layer.parameters()):
        assert torch.equal(a.grad, b.grad)
    if precision == "bf16":
        with torch.no_grad():
            assert torch.equal(pkg.Fp8BlockMoELayer.from_layer(old)(x), pkg.Fp8BlockMoELayer.from_layer(layer)(x))
    pkg.check_status()
