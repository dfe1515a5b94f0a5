"""GPU: products in e4m3 with a scale per block of 128, against 64-bit restatements.

Bounds.  Codes and scales are whole decisions: equal to the bit (a code is the e4m3 value nearest to the real number 448 x / max |x|).  A product
adds K exact products in fp32, each addition off by at most 2^-23 of the sums' size: K 2^-23 sum |x w|, and is rounded to bf16 once, half a step
of 2^-7.  In the experts silu(gate) * up is requantised: where the real number lies closer to the border of two codes than its error, either
code is right, and the result may differ by their distance times the weight; those distances are added up."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn
BF = 2.0 ** -8


def blocks(n):
    return -(-n // 128)


def quant64(x):
    """(codes as float64, scales float64) of rows (N,K)"""
    N, K = x.shape
    p = torch.nn.functional.pad(x.double(), (0, -K % 128)).view(N, -1, 128)
    amax = p.abs().amax(2, keepdim=True).clamp(min=2.0 ** -100)
    codes = (p * 448.0 / amax).clamp(-448, 448).to(F8).double()
    return codes.view(N, -1)[:, :K], (amax[..., 0] / 448.0)


def value64(codes, scale):
    """(..., N, K) codes with their block scales, in 64 bits"""
    N, K = codes.shape[-2:]
    return codes.double() * scale.double().repeat_interleave(128, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]


def rows64(x):
    c, s = quant64(x)
    return c * s.repeat_interleave(128, 1)[:, :x.shape[1]]


def weights(g, *shape, std=0.02):
    w = torch.randn(*shape, generator=g, device=DEV) * std * (0.3 + torch.rand(*shape[:-1], 1, generator=g, device=DEV))
    N, K = shape[-2:]
    s = torch.rand(*shape[:-2], blocks(N), blocks(K), generator=g, device=DEV) * 1e-3 + 1e-4
    full = s.repeat_interleave(128, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]
    return (w / full).clamp(-448, 448).to(F8), s


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.mark.parametrize("N,K", [(1, 8), (3, 128), (5, 136), (700, 1040), (33, 4096), (2000, 264)])
def test_quantisers_bit_exact(pkg, N, K):
    g = gen(N)
    x = (torch.randn(N, K, generator=g, device=DEV) * torch.logspace(-30, 30, N, device=DEV)[:, None]).to(torch.bfloat16)
    x[0, :8] = 0
    if N > 3:
        x[1] = 0
        x[2] = torch.randint(-9, 10, (K,), generator=g, device=DEV).to(torch.bfloat16)     # many values half way between two codes
    q, s = pkg.fp8_block_quantize(x)
    cq, cs = quant64(x)
    assert q.dtype == F8 and torch.equal(q.double(), cq) and torch.equal(s, cs.float())
    w, ws = pkg.fp8_block_quantize_weight(x)
    p = torch.nn.functional.pad(x.double(), (0, -K % 128, 0, -N % 128)).view(blocks(N), 128, blocks(K), 128)
    amax = p.abs().amax((1, 3)).clamp(min=2.0 ** -100)
    cw = (p * 448.0 / amax[:, None, :, None]).clamp(-448, 448).to(F8).double().reshape(blocks(N) * 128, -1)[:N, :K]
    assert torch.equal(w.double(), cw) and torch.equal(ws, (amax / 448).float())
    st, ss = pkg.fp8_block_quantize_weight(torch.stack([x, 2 * x]))
    assert torch.equal(st[0].double(), cw) and torch.equal(ss[1], torch.where(amax > 2.0 ** -100, 2 * ws, ws))      # blocks of zeros have the least scale


def test_quantisers_on_nan_infinity_and_strides(pkg):
    x = torch.randn(6, 256, generator=gen(0), device=DEV).to(torch.bfloat16)
    x[1, 5], x[2, 200] = torch.nan, torch.inf
    q, s = pkg.fp8_block_quantize(x)
    assert torch.isnan(s[1, 0]) and torch.isinf(s[2, 1]) and torch.isfinite(s[[0, 3, 4, 5]]).all()
    v = q.float() * s.repeat_interleave(128, 1)
    assert torch.isnan(v[1, :128]).all() and torch.isnan(v[2, 200]) and torch.isfinite(v[1, 128:]).all() and torch.isfinite(v[2, :128]).all()
    wide = torch.zeros(4, 6, 300, dtype=torch.bfloat16, device=DEV)
    wide[1, :, 3:259] = x
    q2, s2 = pkg.fp8_block_quantize(wide[1, :, 3:259])
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2[[0, 3, 4, 5]], s[[0, 3, 4, 5]])
    e = pkg.fp8_block_quantize(x[:0])
    assert e[0].shape == (0, 256) and e[1].shape == (0, 2)


def check_linear(pkg, M, N, K, seed, grad=True):
    g = gen(seed)
    x = (torch.randn(M, K, generator=g, device=DEV) * (0.1 + torch.rand(M, 1, generator=g, device=DEV))).to(torch.bfloat16).requires_grad_(grad)
    w, s = weights(g, N, K)
    y = pkg.fp8_block_linear(x, w, s)
    wv, xv = value64(w, s), rows64(x.detach())
    ref, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    assert y.shape == (M, N) and y.dtype == torch.bfloat16
    bound = BF * ref.abs() + 1.01 * K * 2.0 ** -23 * size
    assert ((y.double() - ref).abs() <= bound).all(), (M, N, K, float(((y.double() - ref).abs() / bound).max()))
    if grad:
        gy = torch.randn(M, N, generator=g, device=DEV).to(torch.bfloat16)
        (gx,) = torch.autograd.grad(y, x, gy)
        gv = rows64(gy)
        ref, size = gv @ wv, gv.abs() @ wv.abs()
        bound = BF * ref.abs() + 1.01 * N * 2.0 ** -23 * size
        assert ((gx.double() - ref).abs() <= bound).all(), (M, N, K, float(((gx.double() - ref).abs() / bound).max()))
    pkg.check_status()


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 127, 129, 200, 256, 257, 300, 513, 1000])
def test_linear_and_its_gradient(pkg, M):
    for n, (N, K) in enumerate([(8, 16), (128, 128), (136, 144), (256, 1024), (680, 1040), (264, 2064), (1000, 400), (2048, 512)]):
        check_linear(pkg, M, N, K, 100 * M + n)


@pytest.mark.parametrize("M,N,K", [(4, 4096, 4096), (1, 256, 14336), (64, 1408, 2048), (2500, 4096, 1408), (8192, 512, 2048)])
def test_linear_at_length(pkg, M, N, K):
    check_linear(pkg, M, N, K, M)


def test_gradient_of_the_linear_map_is_what_differences_give(pkg):
    """For inputs whose values are codes already (whole numbers up to 16, of which 16 occurs in every block: the factor 448 / 16 = 28 keeps them
    exact only where 28 x is an e4m3 value: x in {0, 1, 2, 4, 8, 16}) the map is linear and exact but for its rounding: y(x + d) - y(x)
    equals W d within the roundings of the two results."""
    g = gen(3)
    pick = torch.tensor([0.0, 1.0, 2.0, 4.0, 8.0, -1.0, -2.0, -4.0], device=DEV)
    x = pick[torch.randint(0, 8, (40, 256), generator=g, device=DEV)]
    x[:, ::128] = 16
    w, s = weights(g, 96, 256)
    d = torch.zeros_like(x)
    d[:, 7] = torch.where(x[:, 7] == 1, 1.0, 0.0)
    y0, y1 = (pkg.fp8_block_linear(t.to(torch.bfloat16), w, s).double() for t in (x, x + d))
    xr = x.to(torch.bfloat16).requires_grad_(True)
    gy = torch.zeros(40, 96, device=DEV)
    gy[:, 5] = 448.0                                   # its code is exact
    (gx,) = torch.autograd.grad(pkg.fp8_block_linear(xr, w, s), xr, gy.to(torch.bfloat16))
    moved = (x[:, 7] == 1)
    lhs = (y1 - y0)[moved, 5]
    assert moved.any() and ((lhs - gx[moved, 7].double() / 448).abs() <= BF * (y0.abs() + y1.abs())[moved, 5] + BF * lhs.abs() + 1e-6).all()


def test_linear_shapes_strides_streams_and_graphs(pkg):
    g = gen(5)
    w, s = weights(g, 264, 272)
    x = torch.randn(3, 50, 272, generator=g, device=DEV).to(torch.bfloat16)
    ref = pkg.fp8_block_linear(x, w, s)
    assert ref.shape == (3, 50, 264) and pkg.fp8_block_linear(x[0, 0], w, s).shape == (264,)
    assert pkg.fp8_block_linear(x[:, :0], w, s).shape == (3, 0, 264)
    wide = torch.zeros(3, 50, 300, dtype=torch.bfloat16, device=DEV)
    wide[..., 5:277] = x
    assert torch.equal(pkg.fp8_block_linear(wide[..., 5:277], w, s), ref)
    wt = w.view(torch.uint8).t().contiguous().t().view(F8)                       # column by column
    odd = torch.empty(w.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(264, 272)
    odd.copy_(w.view(torch.uint8))                                               # a byte past a boundary
    assert torch.equal(pkg.fp8_block_linear(x, wt, s.t().contiguous().t()), ref) and torch.equal(pkg.fp8_block_linear(x, odd.view(F8), s), ref)
    e = torch.zeros(0, 272, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    assert torch.autograd.grad(pkg.fp8_block_linear(e, w, s).sum(), e)[0].shape == (0, 272)
    # a gradient that is broadcast (stride 0) and one in fp32 products
    xr = x.clone().requires_grad_(True)
    (ga,) = torch.autograd.grad(pkg.fp8_block_linear(xr, w, s).sum(), xr)
    (gb,) = torch.autograd.grad(pkg.fp8_block_linear(xr, w, s), xr, torch.ones_like(ref))
    assert torch.equal(ga, gb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    big = torch.randn(700, 272, generator=g, device=DEV).to(torch.bfloat16)
    want = pkg.fp8_block_linear(big, w, s)
    static, sbig = torch.zeros_like(x).requires_grad_(True), torch.zeros_like(big)
    with torch.cuda.stream(side):
        other = pkg.fp8_block_linear(x, w, s)
        torch.autograd.grad(pkg.fp8_block_linear(static, w, s).sum(), static)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ref)
    graphs = []
    for _ in range(2):                                                            # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = pkg.fp8_block_linear(static, w, s)
            (gr,) = torch.autograd.grad(out.sum(), static)
            ob = pkg.fp8_block_linear(sbig, w, s)
        graphs.append((graph, out, gr, ob))
    with torch.no_grad():
        static.copy_(x)
        sbig.copy_(big)
    for _ in range(2):
        for graph, *_ in graphs:
            graph.replay()
    for _, out, gr, ob in graphs:
        assert torch.equal(out, ref) and torch.equal(gr, ga) and torch.equal(ob, want)
    pkg.check_status()


def test_linear_keeps_bad_rows_to_themselves(pkg):
    g = gen(6)
    w, s = weights(g, 256, 512)
    for M in (40, 600):
        x = torch.randn(M, 512, generator=g, device=DEV).to(torch.bfloat16)
        ref = pkg.fp8_block_linear(x, w, s)
        bad = x.clone()
        bad[3, 77], bad[M - 1, 300] = torch.nan, torch.inf
        y = pkg.fp8_block_linear(bad, w, s)
        keep = [i for i in range(M) if i not in (3, M - 1)]
        assert torch.equal(y[keep], ref[keep]) and torch.isnan(y[3]).all() and torch.isnan(y[M - 1]).all()


# ------------------------------------------------------------------------------------------------ experts
def experts64(x, idx, w, gu, gs, dn, ds):
    """(result, bound) in 64 bits"""
    T, H = x.shape
    E, twoI, _ = gu.shape
    I = twoI // 2
    out, bound = torch.zeros(T, H, dtype=torch.float64, device=x.device), torch.zeros(T, H, dtype=torch.float64, device=x.device)
    xv = rows64(x)
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        wv, dv = value64(gu[e], gs[e]), value64(dn[e], ds[e])
        h, eh = xv[t] @ wv.t(), 1.01 * H * 2.0 ** -23 * (xv[t].abs() @ wv.abs().t())
        gate, up, eg, eu = h[:, :I], h[:, I:], eh[:, :I], eh[:, I:]
        a = torch.nn.functional.silu(gate)
        # silu's slope is below 1.1; exponential and quotient of fp32: (2 + 1.17 |gate| + 2 + 2) steps of 2^-23
        v, ev = a * up, 1.1 * eg * up.abs() + a.abs() * eu + 1.1 * eg * eu + (8 + 1.17 * gate.abs()) * 2.0 ** -23 * (a * up).abs()
        b, eb = v.view(len(t), -1, 128), ev.view(len(t), -1, 128)
        amax = b.abs().amax(2, keepdim=True).clamp(min=2.0 ** -100)
        off = eb.amax(2, keepdim=True) / amax + 2.0 ** -22
        q = b * 448.0 / amax
        eq = 448.0 * eb / amax + q.abs() * off
        code = lambda z: z.clamp(-448, 448).to(F8).double()        # noqa: E731
        mid, lo, hi = code(q), code(q - eq), code(q + eq)
        scale = amax / 448.0
        d = (torch.maximum(hi - mid, mid - lo) * scale + mid.abs() * scale * off).view(len(t), I)
        hv = (mid * scale).view(len(t), I)
        y = hv @ dv.t()
        ey = d @ dv.abs().t() + 1.01 * I * 2.0 ** -23 * (hv.abs() @ dv.abs().t()) + BF * y.abs()
        wt = w[t, j].double()[:, None]
        out.index_add_(0, t, wt * y)
        bound.index_add_(0, t, wt.abs() * (ey + BF * ey + 2.0 ** -22 * y.abs()))
    return out, bound + BF * (out.abs() + bound)


def picks(g, T, E, k, how):
    if how == "one":                     # every token's first pick is expert E - 1
        idx = torch.rand(T, E, generator=g, device=DEV)
        idx[:, E - 1] = 2
        return torch.topk(idx, k, dim=1).indices
    z = torch.randn(T, E, generator=g, device=DEV)
    if how == "zipf":
        z -= torch.log(torch.arange(1, E + 1, device=DEV).float()) * 1.5
    return torch.topk(z, k, dim=1).indices


@pytest.mark.parametrize("how", ["even", "zipf", "one"])
@pytest.mark.parametrize("T,E,H,I,k", [(1, 1, 128, 128, 1), (1, 64, 256, 384, 6), (5, 8, 2048, 128, 2), (40, 8, 256, 256, 2), (100, 8, 384, 256, 3),
                                       (300, 16, 256, 128, 4), (700, 8, 256, 512, 2), (1500, 8, 384, 256, 3), (2000, 3, 128, 1408, 2),
                                       (900, 128, 128, 128, 8), (64, 256, 128, 256, 4)])
def test_experts(pkg, T, E, H, I, k, how):
    g = gen(T + E)
    x = torch.randn(T, H, generator=g, device=DEV).to(torch.bfloat16)
    gu, gs = weights(g, E, 2 * I, H, std=0.1)
    dn, ds = weights(g, E, H, I, std=0.1)
    idx = picks(g, T, E, k, how)
    w = torch.rand(T, k, generator=g, device=DEV)
    out = pkg.moe_fp8_block(x, idx, w, gu, gs, dn, ds)
    pkg.check_status()
    ref, bound = experts64(x, idx, w, gu, gs, dn, ds)
    assert out.shape == (T, H) and ((out.double() - ref).abs() <= bound).all(), float(((out.double() - ref).abs() / bound).max())
    # bounds that mean something
    assert float((out.double() - ref).norm() / ref.norm()) < 5e-3


def test_experts_odd_calls(pkg):
    """The same expert twice, picks that name no expert, no tokens, bf16 weights, a bad row, strides, another stream, two graphs."""
    g = gen(1)
    T, E, H, I, k = 90, 8, 256, 256, 3
    x = torch.randn(T, H, generator=g, device=DEV).to(torch.bfloat16)
    gu, gs = weights(g, E, 2 * I, H, std=0.1)
    dn, ds = weights(g, E, H, I, std=0.1)
    args = (gu, gs, dn, ds)
    idx, w = picks(g, T, E, k, "even"), torch.rand(T, k, generator=g, device=DEV)
    ref = pkg.moe_fp8_block(x, idx, w, *args)
    twice = idx.clone()
    twice[:, 1] = twice[:, 0]
    r, b = experts64(x, twice, w, *args)
    assert ((pkg.moe_fp8_block(x, twice, w, *args).double() - r).abs() <= b).all()
    assert pkg.moe_fp8_block(x[:0], idx[:0], w[:0], *args).shape == (0, H)
    bad = x.clone()
    bad[4, 9] = torch.nan
    y = pkg.moe_fp8_block(bad, idx, w, *args)
    keep = [i for i in range(T) if i != 4]
    assert torch.isnan(y[4]).all() and torch.equal(y[keep], ref[keep])
    wide = torch.zeros(T, H + 8, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:H + 3] = x
    assert torch.equal(pkg.moe_fp8_block(wide[:, 3:H + 3], idx.t().contiguous().t(), w.double(), *args), ref)
    pkg.check_status()
    out = idx.clone()
    out[7, 1], out[8, 0] = E, -1
    dropped = w.clone()
    dropped[7, 1] = dropped[8, 0] = 0
    y = pkg.moe_fp8_block(x, out, w, *args)
    with pytest.raises(RuntimeError, match="expert index"):
        pkg.check_status()
    assert torch.equal(y, pkg.moe_fp8_block(x, idx, dropped, *args))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [pkg.moe_fp8_block(x, idx, w, *args) for _ in range(3)]
    here = [pkg.moe_fp8_block(x, idx, w, *args) for _ in range(3)]        # at the same time
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, ref) for o in other + here)
    static, graphs = torch.zeros_like(x), []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = pkg.moe_fp8_block(static, idx, w, *args)
        graphs.append((graph, o))
    static.copy_(x)
    for graph, _ in graphs + graphs:
        graph.replay()
    assert all(torch.equal(o, ref) for _, o in graphs)
    pkg.check_status()


def test_router_then_experts_and_losses(pkg):
    """The operators as they are used together: hidden states through the group-limited router into 8-bit experts, beside an 8-bit shared
    block; and in training the losses' gradient into the gate through the same logits."""
    g = gen(8)
    T, E, H, I, k = 333, 16, 256, 256, 4
    x = torch.randn(T, H, generator=g, device=DEV).to(torch.bfloat16)
    W = (torch.randn(E, H, generator=g, device=DEV) * 0.06).to(torch.bfloat16)
    bias = torch.randn(E, generator=g, device=DEV) * 0.05
    gu, gs = pkg.fp8_block_quantize_weight((torch.randn(E, 2 * I, H, generator=g, device=DEV) * 0.08).to(torch.bfloat16))
    dn, ds = pkg.fp8_block_quantize_weight((torch.randn(E, H, I, generator=g, device=DEV) * 0.08).to(torch.bfloat16))
    sw, ss = pkg.fp8_block_quantize_weight((torch.randn(H, H, generator=g, device=DEV) * 0.06).to(torch.bfloat16))
    with torch.no_grad():
        idx, w, counts = pkg.fused_group_router(x, W, bias, k, E, 4, 2, return_counts=True)
        out = pkg.moe_fp8_block(x, idx, w, gu, gs, dn, ds) + pkg.fp8_block_linear(x, sw, ss)
    ref, bound = experts64(x, idx, w, gu, gs, dn, ds)
    sv = rows64(x) @ value64(sw, ss).t()
    assert ((out.double() - ref - sv).abs() <= bound + BF * (sv.abs() + (ref + sv).abs()) * 1.02 + 1e-4).all()
    assert int(counts.sum()) == T * k
    xt, Wt = x.clone().requires_grad_(True), W.clone().requires_grad_(True)
    idx, w, logits = pkg.fused_group_router(xt, Wt, None, k, E, 4, 2, "softmax", return_logits=True)
    balance, z = pkg.router_losses(logits, idx)
    shared = pkg.fp8_block_linear(xt, sw, ss)
    gx, gW = torch.autograd.grad(balance + 1e-2 * z + w.sum() * 0.1 + shared.float().mean(), (xt, Wt))
    assert torch.isfinite(gx).all() and torch.isfinite(gW).all() and gW.abs().max() > 0 and gx.abs().max() > 0
    pkg.check_status()


def test_quantised_inside_and_before(pkg):
    """Few rows are quantised by the product itself, more of them by a launch before it: a row's result is the same to the bit."""
    g = gen(7)
    x = torch.randn(32, 2048, generator=g, device=DEV).to(torch.bfloat16)
    x[3] = 0
    x[5, 300] = torch.inf
    w, s = weights(g, 1408, 2048)
    few, more = pkg.fp8_block_linear(x[:16], w, s), pkg.fp8_block_linear(x[:17], w, s)
    assert torch.equal(few.view(torch.int16), more[:16].view(torch.int16))
    gu, gs = weights(g, 8, 768, 2048, std=0.1)
    dn, ds = weights(g, 8, 2048, 384, std=0.1)
    idx = torch.rand(32, 8, generator=g, device=DEV).topk(2, dim=1).indices
    wt = torch.rand(32, 2, generator=g, device=DEV)
    few, more = (pkg.moe_fp8_block(x[:n], idx[:n], wt[:n], gu, gs, dn, ds) for n in (16, 32))
    assert torch.equal(few.view(torch.int16), more[:16].view(torch.int16))


def test_few_rows_captured_and_replayed(pkg):
    """A graph of a product and a block of four rows, replayed on other inputs, gives what plain calls give."""
    g = gen(9)
    w, s = weights(g, 512, 512)
    gu, gs = weights(g, 16, 512, 512, std=0.1)
    dn, ds = weights(g, 16, 512, 256, std=0.1)
    x, idx = torch.zeros(4, 512, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 3, dtype=torch.int64, device=DEV)
    wt = torch.rand(4, 3, generator=g, device=DEV)

    def run():
        return pkg.moe_fp8_block(pkg.fp8_block_linear(x, w, s), idx, wt, gu, gs, dn, ds)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        x.copy_(torch.randn(4, 512, generator=g, device=DEV))
        idx.copy_(torch.rand(4, 16, generator=g, device=DEV).topk(3, dim=1).indices)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, run()) and got.abs().sum() > 0
    pkg.check_status()
