"""GPU: low-rank adapters of many requests, against 64 bits.

Bounds.  The tensor cores add in fp32 and may cut off instead of rounding: a sum of n products is off by n 2^-23 of the products' sizes.  x A^T
(and g B) goes on as two bf16 numbers; most tests here allow for one, 2^-8 of its size, and `test_what_goes_on_holds_sixteen_bits` does not.  The result
is off by half a step of its type more.
What is off in the first product goes through the second: `spread` is its sizes times the sizes of the second factor."""
import importlib

import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
STEP, BF_HALF = 2.0 ** -23, 2.0 ** -8


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def make(T, K, N, R, n, how="mixed", seed=0, base=True, dtype=BF):
    g = gen(seed)
    x = torch.randn(T, K, generator=g, device=DEV).to(BF)
    a = (torch.randn(n, R, K, generator=g, device=DEV) / K ** 0.5).to(dtype)
    b = (torch.randn(n, N, R, generator=g, device=DEV) * 0.3).to(dtype)
    s = 0.5 + torch.rand(n, generator=g, device=DEV)
    bs = torch.randn(T, N, generator=g, device=DEV).to(BF) if base else None
    if how == "one":
        index = None
    elif how == "mixed":
        index = torch.randint(-1, n, (T,), generator=g, device=DEV)
    elif how == "tail":      # prompts, then rows of their own requests
        index = torch.arange(T, device=DEV) * 5 // T
        index[-150:] = torch.arange(150, device=DEV) % n
    elif how == "packed":
        ends = (torch.rand(n, generator=g, device=DEV) * T).long().sort().values
        index = (torch.randperm(n + 1, generator=g, device=DEV) - 1)[torch.searchsorted(ends, torch.arange(T, device=DEV), right=True)]
    else:
        index = torch.full((T,), -1, device=DEV)
    return x, a, b, s, bs, index


def reference(x, a, b, s, bs, index, go=None):
    """The formula by adapters in 64 bits: {name: (value, size of what the bf16 rounding in the middle touches, size of the sums' errors)}"""
    T, N = x.shape[0], b.shape[1]
    x, a, b, s = x.double(), a.to(BF).double(), b.to(BF).double(), s.double()
    index = torch.zeros(T, dtype=torch.int64, device=DEV) if index is None else index
    z = lambda *sh: torch.zeros(*sh, dtype=torch.float64, device=DEV)     # noqa: E731
    y, ym, ys = (z(T, N) for _ in range(3))
    if bs is not None:
        y += bs.double()
        ys += bs.double().abs()
    gx, ga, gb = [[z(*t.shape) for _ in range(3)] for t in (x, a, b)]
    for j in range(a.shape[0]):
        t = (index == j).nonzero().flatten()
        if t.numel() == 0:
            continue
        v, vs = s[j] * x[t] @ a[j].t(), s[j] * x[t].abs() @ a[j].abs().t()
        y[t] += v @ b[j].t()
        ym[t] += v.abs() @ b[j].abs().t()
        ys[t] += vs @ b[j].abs().t()
        if go is not None:
            g = go.double()[t]
            u, us = s[j] * g @ b[j], s[j] * g.abs() @ b[j].abs()
            for out, p, q in ((gx, (u, u.abs(), us), a[j]),):
                for o, m, f in zip(out, p, (q, q.abs(), q.abs())):
                    o[t] = m @ f
            for o, m, f in zip(ga, (u, u.abs(), us), (x[t], x[t].abs(), x[t].abs())):
                o[j] = m.t() @ f
            for o, m, f in zip(gb, (v, v.abs(), vs), (g, g.abs(), g.abs())):
                o[j] = f.t() @ m
    return {"y": (y, ym, ys), "gx": gx, "ga": ga, "gb": gb}


def close(got, ref, terms, rounded=True):
    value, middle, sums = ref
    lim = value.abs() * torch.finfo(got.dtype).eps / 2 + (BF_HALF * 1.01 * middle if rounded else 0) + 2 * (terms + 4) * STEP * sums + 2.0 ** -120
    bad = ~((got.double() - value).abs() <= lim)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), float((got.double() - value).norm() / value.norm()))


SHAPES = [(1, 64, 64, 8, 1, "one"), (1, 4096, 4096, 16, 4, "mixed"), (5, 264, 136, 24, 3, "mixed"), (64, 1024, 2816, 16, 64, "mixed"), (127, 520, 680, 128, 5, "packed"),
          (128, 64, 8, 64, 2, "mixed"), (129, 8, 64, 8, 3, "mixed"), (300, 1040, 680, 8, 3, "packed"), (300, 1040, 680, 16, 40, "mixed"), (512, 2048, 2816, 32, 7, "mixed"),
          (1000, 2048, 1408, 64, 1, "one"), (1000, 512, 520, 128, 3, "packed"), (1000, 512, 520, 128, 3, "mixed"), (777, 4096, 1032, 48, 9, "packed"), (260, 256, 256, 16, 2, "none"),
          (1700, 520, 1032, 16, 200, "mixed"), (900, 264, 136, 128, 60, "mixed"), (3000, 136, 264, 32, 12, "tail"), (20000, 128, 72, 16, 5, "packed"), (40000, 64, 64, 8, 2, "packed"), (2100, 64, 14336, 40, 4, "packed")]


@pytest.mark.parametrize("T,K,N,R,n,how", SHAPES)
@pytest.mark.parametrize("base", [True, False])
def test_forward(pkg, T, K, N, R, n, how, base):
    x, a, b, s, bs, index = make(T, K, N, R, n, how, base=base)
    ref = reference(x, a, b, s, bs, index)["y"]
    y = pkg.lora_linear(x, a, b, index, s, bs)
    close(y, ref, max(K, R))
    kept = pkg.lora_linear(x.clone().requires_grad_(), a, b, index, s, bs)       # as a training step runs it
    close(kept.detach(), ref, max(K, R))
    if index is not None:
        assert torch.equal(pkg.lora_linear(x, a, b, index.int(), s, bs), y)
        none = index < 0
        assert torch.equal(y[none], bs[none] if base else torch.zeros_like(y[none]))
    pkg.check_status()


def test_few_rows_are_not_rounded_in_the_middle(pkg):
    x, a, b, s, bs, index = make(100, 1024, 512, 32, 6, base=False)
    close(pkg.lora_linear(x, a, b, index, s), reference(x, a, b, s, None, index)["y"], 1024, rounded=False)


@pytest.mark.parametrize("R", [8, 16, 32, 48, 64, 128])
@pytest.mark.parametrize("how,n", [("one", 1), ("mixed", 3)])
@pytest.mark.parametrize("T", [20, 300])
def test_what_goes_on_holds_sixteen_bits(pkg, T, R, how, n):
    """x A^T and g B are two bf16 numbers, the second off by 2^-8 of at most 2^-8 of the value, on row tiles and with a gradient too.  Short sums, so that
    their bounds are far below what one rounded number would be off."""
    x, a, b, s, _, index = make(T, 16, 24, R, n, how, seed=11, base=False, dtype=F32)
    go = torch.randn(T, 24, generator=gen(12), device=DEV).to(BF)
    leaves = [t.requires_grad_() for t in (x, a, b)]
    y = pkg.lora_linear(x, a, b, index, s)
    got = {"y": y.detach(), **dict(zip(("gx", "ga", "gb"), torch.autograd.grad(y, leaves, go)))}
    ref = reference(x.detach(), a.detach(), b.detach(), s, None, index, go)
    for name, terms in (("y", R), ("gx", R), ("ga", T), ("gb", T)):
        value, middle, sums = ref[name]
        close(got[name], (value, middle * 2.0 ** -8, sums), terms)
    pkg.check_status()


@pytest.mark.parametrize("T,K,N,R,n,how", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradients(pkg, T, K, N, R, n, how, dtype):
    x, a, b, s, bs, index = make(T, K, N, R, n, how, seed=1, dtype=dtype)
    go = torch.randn(T, N, generator=gen(2), device=DEV).to(BF)
    leaves = [t.requires_grad_() for t in (x, a, b, bs)]
    y = pkg.lora_linear(x, a, b, index, s, bs)
    gx, ga, gb, gbase = torch.autograd.grad(y, leaves, go)
    ref = reference(x.detach(), a.detach(), b.detach(), s, bs.detach(), index, go)
    assert gx.dtype == BF and ga.dtype == gb.dtype == dtype and torch.equal(gbase, go)
    close(gx, ref["gx"], max(N, R))
    close(ga, ref["ga"], max(N, T))
    close(gb, ref["gb"], max(K, T))
    if index is not None:
        gone = ~(index[:, None] == torch.arange(n, device=DEV)).any(0)
        assert (ga[gone] == 0).all() and (gb[gone] == 0).all() and (gx[index < 0] == 0).all()
    again = torch.autograd.grad(pkg.lora_linear(x, a, b, index, s, bs), leaves, go)
    assert all(torch.equal(p, q) for p, q in zip((gx, ga, gb, gbase), again))
    # each by itself
    for i, want in enumerate((gx, ga, gb)):
        args = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, a, b))]
        assert torch.equal(torch.autograd.grad(pkg.lora_linear(*args, index, s), args[i], go)[0], want)
    pkg.check_status()


def test_gradient_against_differences(pkg):
    """The result is linear in x and in each factor, so a difference quotient of the forward has no error of its own: the forward's bound over the step."""
    T, K, N, R, n = 150, 128, 64, 16, 3
    x, a, b, s, bs, index = make(T, K, N, R, n, "packed", seed=5)
    go = torch.randn(T, N, generator=gen(6), device=DEV).to(BF)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    grads = torch.autograd.grad(pkg.lora_linear(*leaves, index, s, bs), leaves, go)
    for i in range(3):
        u = torch.randn(leaves[i].shape, generator=gen(7 + i), device=DEV).to(BF) * 4
        ends = [[(t.double() + sign * u.double()).to(BF) if i == j else t for j, t in enumerate((x, a, b))] for sign in (1, -1)]
        moved = (ends[0][i].double() - ends[1][i].double())
        out, room = [], 0.0
        for e in ends:
            out.append(pkg.lora_linear(*e, index, s, bs).double())
            value, middle, sums = reference(*e, s, bs, index)["y"]
            room += float(((value.abs() + middle) * BF_HALF * 1.01 + 300 * STEP * sums).mul(go.double().abs()).sum())
        along = float((grads[i].double() * moved).sum())
        rounding = float((grads[i].double() * moved).abs().sum()) * 2 * BF_HALF
        assert abs(float(((out[0] - out[1]) * go.double()).sum()) - along) <= room + rounding


def test_others_do_not_matter(pkg):
    """NaN and infinity in rows without an adapter, in adapters that no row has and in those of other rows change nothing elsewhere: not the result, not
    the gradients."""
    for T, keep in ((100, False), (500, True)):
        x, a, b, s, bs, _ = make(T, 256, 136, 16, 5)
        index = torch.arange(T, device=DEV) * 7 % 5 - 1          # -1, 0 ... 3; adapter 4 has no row
        go = torch.randn(T, 136, generator=gen(3), device=DEV).to(BF)

        def run(x, a, b, go):
            args = [t.clone().requires_grad_(keep) for t in (x, a, b)]
            y = pkg.lora_linear(*args, index, s, bs)
            return [y.detach(), *(torch.autograd.grad(y, args, go) if keep else ())]

        want = run(x, a, b, go)
        x2, a2, b2, go2 = x.clone(), a.clone(), b.clone(), go.clone()
        bad = float("nan")
        x2[index < 0], a2[4], b2[4], a2[2, 3], b2[2, 5, 7], go2[index < 0] = bad, float("inf"), bad, bad, float("inf"), float("-inf")
        got = run(x2, a2, b2, go2)
        rows = index != 2
        assert torch.equal(got[0][rows], want[0][rows]) and not torch.isfinite(got[0][~rows]).any(1).all()
        if keep:
            others = [0, 1, 3, 4]
            assert torch.equal(got[1][rows], want[1][rows]) and torch.equal(got[2][others], want[2][others]) and torch.equal(got[3][others], want[3][others])
        x3 = x.clone()
        x3[3] = bad          # of adapter index[3]
        got = run(x3, a, b, go)
        rows = torch.arange(T, device=DEV) != 3
        assert torch.equal(got[0][rows], want[0][rows])
        if keep:
            others = [j for j in range(5) if j != int(index[3])]
            assert torch.equal(got[1], want[1]) and torch.equal(got[2][others], want[2][others]) and torch.equal(got[3][others], want[3][others])
    pkg.check_status()


def test_bad_index(pkg):
    for T in (20, 300):
        x, a, b, s, bs, index = make(T, 64, 64, 8, 3)
        bad = index.clone()
        bad[5], bad[T - 1] = 3, 1 << 40
        index[5] = index[T - 1] = -1
        y = pkg.lora_linear(x, a, b, bad, s, bs)
        with pytest.raises(RuntimeError, match="adapter"):
            pkg.check_status()
        assert torch.equal(y, pkg.lora_linear(x, a, b, index, s, bs))
        bad[5], bad[T - 1] = -7, -(1 << 40)
        assert torch.equal(y, pkg.lora_linear(x, a, b, bad, s, bs))
        pkg.check_status()


@pytest.mark.parametrize("T", [40, 260])
def test_layouts(pkg, T):
    K, N, R, n = 264, 136, 16, 3
    x, a, b, s, bs, index = make(T, K, N, R, n)
    want = pkg.lora_linear(x, a, b, index, s, bs)
    wide = torch.randn(T, 3 * K + 8, generator=gen(3), device=DEV).to(BF)
    for view in (wide[:, K:2 * K], wide[:, 3:3 + K], wide[:, : 2 * K : 2], wide.t().contiguous().t()[:, :K], wide[0, :K].expand(T, K)):
        view.copy_(x) if view.stride(0) else None
        plain = view.contiguous()
        assert torch.equal(pkg.lora_linear(view, a, b, index, s, bs), pkg.lora_linear(plain, a, b, index, s, bs))
        leaf = view.detach().requires_grad_()
        dense = plain.clone().requires_grad_()
        g1 = torch.autograd.grad(pkg.lora_linear(leaf, a, b, index, s).float().sum(), leaf)[0]
        g2 = torch.autograd.grad(pkg.lora_linear(dense, a, b, index, s).float().sum(), dense)[0]
        assert torch.equal(g1, g2)
    room = torch.randn(T, 2 * N + 4, generator=gen(4), device=DEV).to(BF)
    for view in (room[:, :N], room[:, 4:4 + N], room[:, 1 : 1 + N]):
        view.copy_(bs)
        assert torch.equal(pkg.lora_linear(x, a, b, index, s, view), want)
    assert torch.equal(pkg.lora_linear(x.view(2, -1, K), a.transpose(1, 2).contiguous().transpose(1, 2), b, index.view(2, -1), s, bs.view(2, -1, N)), want.view(2, -1, N))
    assert torch.equal(pkg.lora_linear(x, a, b, torch.stack([index, index], 1)[:, 0], s, bs), want)
    assert torch.equal(pkg.lora_linear(x[0], a, b, index[0], s, bs[0]), pkg.lora_linear(x[:1], a, b, index[:1], s, bs[:1])[0])
    assert torch.equal(pkg.lora_linear(x, a[:1], b[:1], scaling=2), pkg.lora_linear(x, a[:1], b[:1], torch.zeros(T, dtype=torch.int32, device=DEV), torch.full((1,), 2.0, device=DEV)))
    shared = a[:1].expand(n, R, K).clone()
    one = a[:1].clone().requires_grad_()
    pkg.lora_linear(x, one.expand(n, R, K), b, index, s).float().sum().backward()       # a factor that adapters share
    each = shared.requires_grad_()
    pkg.lora_linear(x, each, b, index, s).float().sum().backward()
    assert torch.equal(one.grad, each.grad.sum(0, keepdim=True))
    pkg.check_status()


def test_empty(pkg):
    x, a, b, s, bs, index = make(0, 64, 72, 8, 3)
    leaves = [t.requires_grad_() for t in (x, a, b, bs)]
    y = pkg.lora_linear(x, a, b, index, s, bs)
    assert y.shape == (0, 72)
    y.sum().backward()
    assert [t.grad.shape for t in leaves] == [t.shape for t in leaves] and (a.grad == 0).all() and (b.grad == 0).all()
    x, a, b, s, bs, index = make(30, 64, 72, 8, 3)
    assert torch.equal(torch.autograd.grad(pkg.lora_linear(x, a, b, index, s, bs.requires_grad_()), bs, x.new_ones(30, 72))[0], x.new_ones(30, 72))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g = torch.autograd.grad(pkg.lora_linear(x.requires_grad_(), a, b, index, s).float().square().sum(), x, create_graph=True)[0]
        g.float().sum().backward()


@pytest.mark.parametrize("T", [16, 700])
def test_streams_and_graphs(pkg, T):
    x, a, b, s, bs, index = make(T, 512, 264, 16, 4, "packed")
    go = torch.randn(T, 264, generator=gen(5), device=DEV).to(BF)

    def step(x, a, b):
        y = pkg.lora_linear(x, a, b, index, s, bs)
        with torch.no_grad():
            quiet = pkg.lora_linear(x, a, b, index, s, bs)
        return [y.detach(), quiet, *torch.autograd.grad(y, [x, a, b], go)]

    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    want = [t.clone() for t in step(*leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step(*leaves)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*leaves))
    with torch.no_grad():
        for t, seed in zip(leaves, (11, 12, 13)):
            t.copy_((torch.randn(t.shape, generator=gen(seed), device=DEV) * 0.1).to(BF))
        index.copy_(index.roll(T // 3))
    for g in graphs:
        g.replay()
    want = step(*leaves)
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))
    pkg.check_status()


@pytest.mark.parametrize("T", [30, 200, 900])
def test_inference_mode_and_two_calls_at_once(pkg, T):
    """Calls on two streams at a time have workspaces of their own."""
    x, a, b, s, bs, index = make(T, 512, 264, 16, 6)
    x2, a2, b2, s2, bs2, index2 = make(T, 1024, 520, 32, 9, seed=4)
    want, want2 = pkg.lora_linear(x, a, b, index, s, bs), pkg.lora_linear(x2, a2, b2, index2, s2, bs2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    with torch.inference_mode():
        for _ in range(10):
            with torch.cuda.stream(streams[0]):
                got[0].append(pkg.lora_linear(x, a, b, index, s, bs))
            with torch.cuda.stream(streams[1]):
                got[1].append(pkg.lora_linear(x2, a2, b2, index2, s2, bs2))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got[0]) and all(torch.equal(o, want2) for o in got[1])
    pkg.check_status()


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traced_forward_gradients_and_autocast(pkg):
    x, a, b, s, bs, index = make(40, 256, 64, 16, 3)
    fn = lambda x, index: pkg.lora_linear(x, a, b, index, s)      # noqa: E731
    with torch.no_grad():
        traced = torch.jit.trace(fn, (x, index))
        for T in (40, 7, 300):
            x2, _, _, _, _, i2 = make(T, 256, 64, 16, 3, seed=T)
            assert torch.equal(traced(x2, i2), fn(x2, i2))
    with fw.dual_level(), pytest.raises(Exception, match="forward"):
        fn(fw.make_dual(x, torch.ones_like(x)), index)
    with torch.autocast("cuda", dtype=BF):
        assert torch.equal(pkg.lora_linear(x.float(), a.float(), b.float(), index, s, bs.float()), pkg.lora_linear(x, a, b, index, s, bs))


def test_observer(pkg):
    x, a, b, s, bs, index = make(3000, 256, 64, 16, 3)

    def seen(call):
        names = []
        pkg.ops.set_hook(lambda name, launches, p, q: names.append((name, launches)))
        try:
            call()
        finally:
            pkg.ops.set_hook(None)
        torch.cuda.synchronize()
        return names

    assert seen(lambda: pkg.lora_linear(x[:4], a, b, index[:4], s)) == [("lora_few", 1)]
    assert seen(lambda: pkg.lora_linear(x, a, b, index, s)) == [("lora_tiles", 1), ("lora_shrink", 1), ("lora_expand", 1)]
    assert seen(lambda: pkg.lora_linear(x, a[:1], b[:1])) == [("lora_shrink", 1), ("lora_expand", 1)]
    x.requires_grad_(), a.requires_grad_(), b.requires_grad_()
    got = [n for n, _ in seen(lambda: pkg.lora_linear(x, a, b, index, s).float().sum().backward())]
    assert sorted(got) == sorted(["lora_tiles", "lora_shrink", "lora_expand", "lora_back", "lora_expand", "lora_wgrad"])


def test_refusals(pkg):
    x, a, b, s, bs, index = make(4, 64, 72, 8, 3)
    for match, call in (("bfloat16", lambda: pkg.lora_linear(x.float(), a, b, index)), ("both", lambda: pkg.lora_linear(x, a, b.float(), index)),
                        ("agree", lambda: pkg.lora_linear(x, a[:2], b, index)), ("rank", lambda: pkg.lora_linear(x, a[:, :4], b[..., :4], index)),
                        ("rank", lambda: pkg.lora_linear(x, a.repeat(1, 17, 1), b.repeat(1, 1, 17), index)), ("x must be", lambda: pkg.lora_linear(x[:, :8], a, b, index)),
                        ("without an index", lambda: pkg.lora_linear(x, a, b)), ("index must be", lambda: pkg.lora_linear(x, a, b, index[:2])),
                        ("index must be", lambda: pkg.lora_linear(x, a, b, index.float())), ("scaling", lambda: pkg.lora_linear(x, a, b, index, s[:2])),
                        ("scaling takes no gradient", lambda: pkg.lora_linear(x, a, b, index, s.clone().requires_grad_())),
                        ("base must be", lambda: pkg.lora_linear(x, a, b, index, s, bs[:, :64])), ("multiples of 8", lambda: pkg.lora_linear(x[:, :12], a[..., :12], b, index))):
        with pytest.raises(ValueError, match=match):
            call()


def test_beside_a_frozen_product(pkg):
    """As they are used: norm, the product of its codes, the adapters on its rows; forward and backward against the steps taken one by one in 64 bits on
    the same codes, and served."""
    T, K, N, R, n = 300, 1040, 680, 16, 3
    x, a, b, s, _, index = make(T, K, N, R, n, "packed")
    g = gen(9)
    r = torch.randn(T, K, generator=g, device=DEV).to(BF)
    wn = (1 + 0.1 * torch.randn(K, generator=g, device=DEV)).to(BF)
    w, ws = pkg.fp8_block_quantize_weight((torch.randn(N, K, generator=g, device=DEV) * 0.05).to(BF))
    leaves = [t.requires_grad_() for t in (x, r, wn, a, b)]
    q, qs, y, h = pkg.rms_norm_fp8_block(x, wn, r, return_norm=True)
    product = pkg.fp8_block_linear(y, w, ws, quantized=(q, qs))
    out = pkg.lora_linear(y, a, b, index, s, base=product)
    ref = reference(y.detach(), a.detach(), b.detach(), s, product.detach(), index)["y"]
    close(out.detach(), ref, K)
    go, gh = (torch.randn(T, m, generator=g, device=DEV).to(BF) for m in (N, K))
    got = torch.autograd.grad([out, h], leaves, [go, gh])
    y2 = y.detach().requires_grad_()
    through = torch.autograd.grad(pkg.lora_linear(y2, a, b, index, s), [y2, a, b], go)
    frozen = torch.autograd.grad(pkg.fp8_block_linear(y2, w, ws), y2, go)[0]
    want = torch.autograd.grad(pkg.rms_norm(x, wn, r), [x, r, wn], [through[0] + frozen, gh])
    assert all(torch.equal(p, q) for p, q in zip(got, (*want, *through[1:])))
    with torch.no_grad():
        for m in (1, 16, 100, T):
            q, qs, y, h = pkg.rms_norm_fp8_block(x[:m], wn, r[:m], return_norm=True)
            served = pkg.lora_linear(y, a, b, index[:m], s, base=pkg.fp8_block_linear(None, w, ws, quantized=(q, qs)))
            close(served, tuple(t[:m] for t in ref), K, rounded=True)
    pkg.check_status()


def test_first_call_of_a_thread(pkg):
    """A thread that has not touched the GPU before (the autograd engine's, or a user's) calls the kernels as its first act."""
    import threading
    x, a, b, s, bs, index = make(300, 64, 64, 8, 3)
    want = pkg.lora_linear(x, a, b, index, s, bs)
    out = torch.empty_like(want)
    lib, L = pkg.lib(), importlib.import_module(pkg.__name__ + "._lib")
    ws = L.workspace(lib.b200moe_lora_fwd_ws_bytes(300, 8, 3, 0), x.device)
    args = (x.data_ptr(), 64, a.data_ptr(), b.data_ptr(), index.data_ptr(), 8, s.data_ptr(), 1.0, bs.data_ptr(), 64, 300, 64, 64, 8, 3, 0, ws.data_ptr(), out.data_ptr(),
            L.status_word(x.device).data_ptr(), L.stream_of(x))
    rc = []
    t = threading.Thread(target=lambda: rc.append(lib.b200moe_lora_forward(*args)))
    t.start()
    t.join()
    L.check(rc[0])
    assert torch.equal(out, want)


@pytest.mark.parametrize("T", [40, 700])
def test_rows_of_a_larger_batch(pkg, T):
    """Everything a slice from the second row on: int32 indices lie at no multiple of eight bytes then."""
    x, a, b, s, bs, index = make(T + 1, 64, 72, 16, 3, seed=21)
    want = pkg.lora_linear(x[1:].clone(), a, b, index[1:].clone(), s, bs[1:].clone())
    for i in (index[1:], index.int()[1:]):
        assert torch.equal(pkg.lora_linear(x[1:], a, b, i, s, bs[1:]), want)
    n = torch.stack([index, index], 1).int()[:, 1]      # and every second of them
    assert torch.equal(pkg.lora_linear(x, a, b, n, s, bs), pkg.lora_linear(x, a, b, index, s, bs))
    pkg.check_status()


def test_offsets_beyond_32_bits(pkg):
    """x, base, the result and both gradients have more than 2^31 values; only the last rows have a gradient, so those are all that the sums hold."""
    T, K, N, R, n, m = 270_000, 8192, 8200, 16, 3, 1000
    x, bs = (torch.empty(T, d, dtype=BF, device=DEV).normal_(generator=gen(31)) for d in (K, N))
    _, a, b, s, _, _ = make(1, K, N, R, n, seed=32)
    go = torch.zeros(T, N, dtype=BF, device=DEV)
    go[-m:].normal_(generator=gen(33))
    for index in (torch.arange(T, device=DEV) * n // T, torch.arange(T, device=DEV) * 7 % (n + 1) - 1):
        leaves = [t.requires_grad_() for t in (x, a, b)]
        y = pkg.lora_linear(x, a, b, index, s, bs)
        gx, ga, gb = torch.autograd.grad(y, leaves, go)
        ref = reference(x.detach()[-m:], a.detach(), b.detach(), s, bs[-m:], index[-m:], go[-m:])
        close(y.detach()[-m:], ref["y"], K)
        close(gx[-m:], ref["gx"], N)
        close(ga, ref["ga"], N)
        close(gb, ref["gb"], K)
        del y, gx
    pkg.check_status()
