"""GPU: the operators behind the layers: `MoELayer` with groups of experts, softmax scores and the routers' losses, and `Fp8BlockMoELayer`."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(pkg, **kw):
    torch.manual_seed(0)
    return pkg.MoELayer(256, 128, 16, top_k=3, **kw).to(DEV).to(torch.bfloat16)


def hidden(*shape):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)


@pytest.mark.parametrize("kw", [dict(num_groups=4, topk_groups=2), dict(scoring="softmax", balance_loss=0.5, z_loss=0.25),
                                dict(scoring="softmax", num_groups=4, topk_groups=1, group_score="max", precision="mxfp8", z_loss=0.1),
                                dict(balance_loss=1.0, balance_per_sequence=True, act_codes=[0, 1, 5, 0] * 4)])
def test_layer_is_its_parts(pkg, kw):
    """Output, losses and gradients of a layer are those of router, losses and experts called one by one: the same bits."""
    layer = make(pkg, **kw)
    with torch.no_grad():
        layer.bias.copy_(torch.linspace(-0.02, 0.02, 16, device=DEV))
    x = hidden(3, 50, 256).requires_grad_(True)
    go = hidden(3, 50, 256)
    mask = torch.arange(50, device=DEV)[None] < torch.tensor([[50], [20], [0]], device=DEV) if layer.balance_loss or layer.z_loss else None
    out = layer(x, mask)
    params = [x, layer.gate.weight, layer.gate_up_proj, layer.down_proj]
    aux = layer.aux_loss
    assert (aux is not None) == bool(layer.balance_loss or layer.z_loss)
    got = torch.autograd.grad((out.float() * go.float()).sum() + (0 if aux is None else 3 * aux), params)
    idx, w, counts, logits = pkg.fused_group_router(x, layer.gate.weight, layer.bias, 3, 16, layer.num_groups, layer.topk_groups, layer.scoring,
                                                    layer.group_score, return_counts=True, return_logits=True)
    fn = pkg.moe_mxfp8 if layer.precision == "mxfp8" else pkg.moe
    ref = fn(x.reshape(-1, 256), idx.reshape(-1, 3), w.reshape(-1, 3), layer.gate_up_proj, layer.down_proj, layer.act_codes).view(3, 50, 256)
    total = (ref.float() * go.float()).sum()
    if aux is not None:
        balance, z = pkg.router_losses(logits, idx, layer.scoring, mask, layer.balance_per_sequence)
        total = total + 3 * (layer.balance_loss * balance + layer.z_loss * z)
        assert torch.equal(aux, layer.balance_loss * balance + layer.z_loss * z) and float(aux.detach()) > 0
    assert torch.equal(out, ref) and torch.equal(layer.last_counts, counts)
    for a, b in zip(got, torch.autograd.grad(total, params)):
        assert torch.equal(a, b)
    if layer.num_groups == 4:
        assert all(len(set((r // 4).tolist())) <= layer.topk_groups for r in idx.view(-1, 3)[:40].cpu())
    before = layer.bias.clone()
    layer.update_bias(1e-3)
    assert not torch.equal(before, layer.bias) and int(layer._load_tensor().sum()) == 0
    layer.eval()
    assert layer(x.detach()).shape == x.shape and layer.aux_loss is None
    pkg.check_status()


def test_a_plain_layer_is_what_it_was(pkg):
    a, b = make(pkg), make(pkg)
    x = hidden(70, 256)
    assert torch.equal(a(x), b(x)) and a.aux_loss is None
    with pytest.raises(ValueError, match="mask"):
        a(x, torch.ones(70, device=DEV))
    with pytest.raises(ValueError, match="groups"):
        make(pkg, num_groups=5)(x)
    with pytest.raises(ValueError, match="scoring"):
        make(pkg, scoring="tanh")(x)


def test_a_layer_is_copied_after_a_training_forward(pkg):
    layer = make(pkg, scoring="softmax", balance_loss=0.1)
    x = hidden(70, 256)
    out = layer(x)
    other = copy.deepcopy(layer)
    assert other.aux_loss is None and layer.aux_loss is not None and torch.equal(other(x), out)
    layer.aux_loss.backward()
    assert layer.gate.weight.grad is not None


def test_losses_balance_the_router(pkg):
    """A training step captured into a graph, its losses among it, gives what the same step gives outside."""
    layer = make(pkg, scoring="softmax", balance_loss=0.1, z_loss=0.01)
    x, static = hidden(64, 256), torch.zeros(64, 256, dtype=torch.bfloat16, device=DEV)
    params = [p for p in layer.parameters()]

    def step(inp):
        out = layer(inp)
        return torch.autograd.grad(out.float().square().mean() + layer.aux_loss, params)

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(static)
    static.copy_(x)
    graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kw", [{}, dict(num_groups=4, topk_groups=2), dict(scoring="softmax")])
def test_fp8_layer(pkg, kw):
    layer = make(pkg, **kw).eval()
    with torch.no_grad():
        layer.bias.copy_(torch.linspace(-0.02, 0.02, 16, device=DEV))
    q = pkg.Fp8BlockMoELayer.from_layer(layer)
    x = hidden(2, 40, 256)
    out = q(x)
    assert out.shape == x.shape and not out.requires_grad and not any(p.requires_grad for p in q.parameters())
    flat = x.view(-1, 256)
    if kw:
        idx, w = pkg.fused_group_router(flat, layer.gate.weight, layer.bias, 3, 16, layer.num_groups, layer.topk_groups, layer.scoring)
    else:
        idx, w = pkg.fused_mlp_router(flat, layer.gate.weight, layer.bias, 3, 16)
    with torch.no_grad():
        assert torch.equal(out.view(-1, 256), pkg.moe_fp8_block(flat, idx, w, q.gate_up_proj, q.gate_up_scale, q.down_proj, q.down_scale))
        # e4m3 has steps of 2^-3 to 2^-4 of a value, off by half a step: 4 % at most, 2.5 % in the mean square, of x, W, inter and W again, and
        # through the product gate * up twice for the first two: sqrt(2 * 2 + 2) * 2.5 % = 6 %; 12 % is twice that
        ref = layer(x)
    assert float((out.float() - ref.float()).norm() / ref.float().norm()) < 0.12
    # a state dict, a cast and a move keep codes and scales
    fresh = pkg.Fp8BlockMoELayer(256, 128, 16, top_k=3, **kw).to(DEV)
    fresh.load_state_dict(q.state_dict())
    fresh.to(torch.bfloat16).to(torch.float16).to(torch.bfloat16)
    assert fresh.gate_up_proj.dtype == torch.float8_e4m3fn and fresh.down_scale.dtype == torch.float32 and fresh.bias.dtype == torch.float32
    fresh.gate.weight.data = q.gate.weight.data
    assert torch.equal(fresh(x), out)
    moved = fresh.cpu()
    assert moved.gate_up_proj.device.type == "cpu" and moved.gate_up_scale.dtype == torch.float32
    assert q(x[:, :0]).shape == (2, 0, 256)
    with pytest.raises(ValueError, match="multiples of 128"):
        pkg.Fp8BlockMoELayer(200, 128, 4)
    with pytest.raises(ValueError, match="SiLU-GLU"):
        pkg.Fp8BlockMoELayer.from_layer(make(pkg, act_codes=[1] * 16))
