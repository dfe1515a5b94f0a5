"""GPU: calls of the adapters that take tiles of 128 rows, and that they do; and few rows with clusters of four.  Bounds as in tests/test_gpu_lora.py."""
import importlib
import threading

import pytest
import torch

from .test_gpu_lora import BF, DEV, close, gen, make, reference
from .test_gpu_reserved_sms import grids

pytestmark = pytest.mark.gpu
TILES = ["lora_tiles", "lora_shrink", "lora_expand"]


def launched(pkg, call):
    """What a call gives, and the operations that it queues"""
    names = []
    pkg.ops.set_hook(lambda name, launches, p, q: names.append(name))
    try:
        out = call()
    finally:
        pkg.ops.set_hook(None)
    torch.cuda.synchronize()
    return out, names


def test_first_call_of_a_thread(pkg):
    """Tensor maps are encoded in a thread that has not touched the GPU before."""
    T = 700
    x, a, b, s, bs, index = make(T, 64, 64, 8, 3)
    want, names = launched(pkg, lambda: pkg.lora_linear(x, a, b, index, s, bs))
    assert names == TILES
    out = torch.empty_like(want)
    lib, L = pkg.lib(), importlib.import_module(pkg.__name__ + "._lib")
    ws = L.workspace(lib.b200moe_lora_fwd_ws_bytes(T, 8, 3, 0), x.device)
    args = (x.data_ptr(), 64, a.data_ptr(), b.data_ptr(), index.data_ptr(), 8, s.data_ptr(), 1.0, bs.data_ptr(), 64, T, 64, 64, 8, 3, 0, ws.data_ptr(), out.data_ptr(),
            L.status_word(x.device).data_ptr(), L.stream_of(x))
    rc = []
    t = threading.Thread(target=lambda: rc.append(lib.b200moe_lora_forward(*args)))
    t.start()
    t.join()
    L.check(rc[0])
    assert torch.equal(out, want)


@pytest.mark.parametrize("T", [20, 300, 700])
def test_bad_index(pkg, T):
    """Rows that name no adapter there is, in the result, in the lists of the gradients and reported by either."""
    x, a, b, s, bs, index = make(T, 64, 72, 8, 3)
    go = torch.randn(T, 72, generator=gen(5), device=DEV).to(BF)
    over, under = index.clone(), index.clone()
    at = [5, T // 2, T - 1]
    over[at] = torch.tensor([3, 1 << 40, 1 << 31], device=DEV)
    under[at] = torch.tensor([-7, -(1 << 40), -(1 << 31)], device=DEV)
    index[at] = -1
    leaves = [t.requires_grad_() for t in (x, a, b)]

    def step(i):
        y = pkg.lora_linear(x, a, b, i, s, bs)
        with torch.no_grad():
            quiet = pkg.lora_linear(x, a, b, i, s, bs)
        return [quiet, y.detach(), *torch.autograd.grad(y, leaves, go)]

    want, names = launched(pkg, lambda: step(index))
    assert ("lora_few" in names) == (T <= 512) and names.count("lora_tiles") == (1 if T <= 512 else 2)
    pkg.check_status()
    for bad, raises in ((over, True), (under, False), (torch.where(over > 2, 3, over).int(), True)):
        got = step(bad)
        if raises:
            with pytest.raises(RuntimeError, match="adapter"):
                pkg.check_status()
        else:
            pkg.check_status()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    with torch.no_grad():          # the forward without a gradient reports by itself
        pkg.lora_linear(x, a, b, over, s, bs)
    with pytest.raises(RuntimeError, match="adapter"):
        pkg.check_status()
    ref = reference(x.detach(), a.detach(), b.detach(), s, bs, index, go)
    for got, name, terms in zip(want[1:], ("y", "gx", "ga", "gb"), (64, 72, T, T)):
        close(got, ref[name], terms)


@pytest.mark.parametrize("T", [700, 1100])
def test_layouts(pkg, T):
    """Rows of x and of the base inside wider ones, read in place where they lie at multiples of 16 bytes."""
    K, N, R, n = 264, 136, 16, 3
    x, a, b, s, bs, index = make(T, K, N, R, n)
    want, names = launched(pkg, lambda: pkg.lora_linear(x, a, b, index, s, bs))
    assert names == TILES
    close(want, reference(x, a, b, s, bs, index)["y"], K)
    room = torch.randn(T, 2 * N + 8, generator=gen(4), device=DEV).to(BF)
    for view in (room[:, :N], room[:, 8:8 + N], room[:, 4:4 + N], room[:, 1:1 + N], room[:, : 2 * N : 2]):
        view.copy_(bs)
        before = room.clone()
        assert torch.equal(pkg.lora_linear(x, a, b, index, s, view), want) and torch.equal(room, before)
    assert torch.equal(pkg.lora_linear(x, a, b, index, s, bs[0].expand(T, N)), pkg.lora_linear(x, a, b, index, s, bs[:1].repeat(T, 1)))
    wide = torch.randn(T, 3 * K + 8, generator=gen(3), device=DEV).to(BF)
    for view in (wide[:, K:2 * K], wide[:, 3:3 + K], wide[:, : 2 * K : 2]):
        view.copy_(x)
        assert torch.equal(pkg.lora_linear(view, a, b, index, s, bs), want)
        assert torch.equal(pkg.lora_linear(view, a, b, index, s, room[:, 8:8 + N].copy_(bs)), want)


# ranks of one step of 16, of two and of more, with as many groups as give clusters of four; rows that are ranked in every CTA (up to 128) and by a kernel before
FOURS = [(300, 520, 680, 16, 60), (300, 520, 680, 24, 60), (300, 1040, 264, 32, 90), (300, 264, 520, 48, 60), (300, 520, 680, 128, 60), (512, 64, 1408, 64, 100),
         (100, 520, 680, 32, 80), (128, 264, 136, 40, 70), (128, 136, 2816, 128, 128), (64, 264, 264, 32, 64)]


@pytest.mark.parametrize("T,K,N,R,n", FOURS)
@pytest.mark.parametrize("base", [True, False])
def test_few_rows_of_many_adapters(pkg, T, K, N, R, n, base):
    x, a, b, s, bs, index = make(T, K, N, R, n, seed=51, base=base)
    y, names = launched(pkg, lambda: pkg.lora_linear(x, a, b, index, s, bs))
    assert names == ["lora_few"]
    steps = 1 if R <= 16 else 2 if R <= 32 else 0
    assert any(f"lora_few_kernelILi{steps}ELi4E" in name for name, _ in grids(lambda: pkg.lora_linear(x, a, b, index, s, bs)))
    value, middle, sums = reference(x, a, b, s, bs, index)["y"]
    close(y, (value, middle * 2.0 ** -8, sums), max(K, R))
    none = index < 0
    assert torch.equal(y[none], bs[none] if base else torch.zeros_like(y[none]))
    assert torch.equal(pkg.lora_linear(x, a, b, index.int(), s, bs), y)
    pkg.check_status()
