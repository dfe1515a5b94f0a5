"""GPU: SMs that are reserved for an exchange (`b200moe_set_reserved_sms`) stay free of the norm and of the adapters' products: their grids, read from a captured graph, fit the others."""
import pytest
import torch
from cuda.bindings import driver

from .test_gpu_lora import BF, DEV, close, gen, make, reference
from .test_gpu_norm import EPS, norm64
from .test_gpu_norm import close as close_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[0, 40, 120, 146])
def sms(pkg, request):
    lib = pkg.lib()
    all_sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    assert lib.b200moe_set_reserved_sms(min(request.param, all_sms - 2)) == 0
    try:
        yield all_sms - min(request.param, all_sms - 2)
    finally:
        assert lib.b200moe_set_reserved_sms(0) == 0


def grids(call):
    """(kernel, CTAs) of what a call launches"""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    handle = driver.CUgraph(graph.raw_cuda_graph())
    ok = driver.CUresult.CUDA_SUCCESS
    err, _, n = driver.cuGraphGetNodes(handle, 0)
    assert err == ok
    err, nodes, n = driver.cuGraphGetNodes(handle, n)
    assert err == ok
    out = []
    for node in nodes[:n]:
        err, kind = driver.cuGraphNodeGetType(node)
        assert err == ok
        if kind != driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            continue
        err, p = driver.cuGraphKernelNodeGetParams(node)
        assert err == ok
        err, name = driver.cuFuncGetName(p.func) if int(p.func) else driver.cuKernelGetName(p.kern)
        assert err == ok
        out.append((name.decode(), p.gridDimX * p.gridDimY * p.gridDimZ))
    return out


def ctas(found, part):
    mine = [n for name, n in found if part in name]
    assert mine, (part, found)
    return max(mine)


def test_adapters(pkg, sms):
    """Of the row tiles' kernels an SM has two CTAs of the first product or one each of the gradient's two, and one of the second."""
    T, K, N, R, n = 3000, 520, 2176, 16, 3
    x, a, b, s, bs, index = make(T, K, N, R, n, "packed", seed=41)
    go = torch.randn(T, N, generator=gen(42), device=DEV).to(BF)
    leaves = [t.requires_grad_() for t in (x, a, b)]
    got = []

    def step():
        y = pkg.lora_linear(x, a, b, index, s, bs)
        got[:] = [y.detach(), *torch.autograd.grad(y, leaves, go)]

    found = grids(step)
    assert ctas(found, "lora_shrink") <= 2 * sms and ctas(found, "lora_expand") <= sms
    # the factors' gradients have a CTA for 128 columns of an adapter at least, and are not persistent; whole clusters, of eight at most
    assert ctas(found, "lora_back") <= sms + max(sms, N // 128 * n) + 7 and ctas(found, "lora_wgrad_kernel") <= max(2 * sms, (K + 127) // 128 * n)
    step()
    ref = reference(x.detach(), a.detach(), b.detach(), s, bs, index, go)
    for t, name, terms in zip(got, ("y", "gx", "ga", "gb"), (max(K, R), max(N, R), max(N, T), max(K, T))):
        close(t, ref[name], terms)
    few = 64
    with torch.no_grad():
        close(pkg.lora_linear(x[:few], a, b, index[:few], s, bs[:few]), tuple(t[:few] for t in ref["y"]), max(K, R))
    pkg.check_status()


@pytest.mark.parametrize("T,K,at_once", [(5000, 2048, 2), (5000, 1037, 16), (4000, 128, 4), (4000, 120, 4), (4000, 121, 4), (100, 4096, 2)])
def test_norm(pkg, sms, T, K, at_once):
    """At most `at_once` CTAs an SM."""
    g = gen(43)
    x, r, gy = (torch.randn(T, K, generator=g, device=DEV).to(BF) for _ in range(3))
    w = (1 + 0.3 * torch.randn(K, generator=g, device=DEV)).to(BF)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    got = []

    def step():
        y, h = pkg.rms_norm(x, w, r, EPS)
        got[:] = [y.detach(), h.detach(), *torch.autograd.grad(y, leaves, gy)]

    found = grids(step)
    assert ctas(found, "rms_norm_fwd") <= at_once * sms and ctas(found, "rms_norm_bwd") <= at_once * sms, found
    step()
    y, h, gx, _, gw = got
    ref, rstd = norm64(h, w.detach())
    n = h.double() * rstd
    d = gy.double() * w.detach().double()
    back = (d * n).mean(-1, keepdim=True)
    close_norm(y, ref, ref.abs(), 2.0 ** -19)
    close_norm(gx, rstd * (d - n * back), rstd * (d.abs() + n.abs() * (d * n).abs().mean(-1, keepdim=True)), 2.0 ** -17)
    close_norm(gw, (gy.double() * n).sum(0), (gy.double() * n).abs().sum(0), 2.0 ** -17)
    pkg.check_status()
