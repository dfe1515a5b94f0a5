"""GPU: adapters in fp32 captured and replayed, recomputed and offloaded; backward passes of two threads at once.  What a call gives does not depend on any of it."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from .test_gpu_lora import BF, DEV, F32, gen, make

pytestmark = pytest.mark.gpu


def start(T, K=264, N=520, R=24, n=3, dtype=F32, seed=61):
    x, a, b, s, bs, index = make(T, K, N, R, n, "packed", seed=seed, dtype=dtype)
    go = torch.randn(T, N, generator=gen(seed + 1), device=DEV).to(BF)
    return [t.requires_grad_() for t in (x, a, b)], index, s, bs, go


@pytest.mark.parametrize("T", [30, 700])
def test_captured(pkg, T):
    leaves, index, s, bs, go = start(T)

    def step():
        y = pkg.lora_linear(*leaves, index, s, bs)
        with torch.no_grad():
            quiet = pkg.lora_linear(*leaves, index, s, bs)
        return [y.detach(), quiet, *torch.autograd.grad(y, leaves, go)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    with torch.no_grad():
        for t, seed in zip(leaves, (11, 12, 13)):
            t.copy_(torch.randn(t.shape, generator=gen(seed), device=DEV) * 0.1)
        index.copy_(index.roll(T // 3))
    for g in graphs:
        g.replay()
    want = step()
    assert want[3].dtype == F32
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))
    pkg.check_status()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_recomputed_and_offloaded(pkg, dtype):
    leaves, index, s, bs, go = start(700, dtype=dtype)
    call = lambda x, a, b: pkg.lora_linear(x, a, b, index, s, bs)     # noqa: E731
    want = torch.autograd.grad(call(*leaves), leaves, go)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves, go), want))
    with torch.autograd.graph.save_on_cpu():
        y = call(*leaves)
    for _ in range(2):
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, go, retain_graph=True), want))
    pkg.check_status()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_two_threads(pkg, dtype):
    work = [start(T, seed=seed, dtype=dtype) for T, seed in ((700, 71), (1300, 81))]
    step = lambda w: torch.autograd.grad(pkg.lora_linear(*w[0], w[1], w[2], w[3]), w[0], w[4])     # noqa: E731
    want = [step(w) for w in work]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                got[i].append(step(work[i]))
        st.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for mine, right in zip(got, want):
        assert len(mine) == 20 and all(torch.equal(p, q) for g in mine for p, q in zip(g, right))
    pkg.check_status()
