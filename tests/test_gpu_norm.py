"""GPU: the root-mean-square norm with residual and 8-bit rows, against 64 bits.

Bounds.  A row's sum of squares goes through at most 32 additions of a thread, 10 of shuffles and a few roundings after: rstd is off by less than
(42 / 2 + 4) 2^-24 < 2^-19, and n, y and the code's factor with it.  What is stored is off by half a step of its type more.  mean(d n) is off by
2^-18 of mean(|d n|), so the gradient's two terms by 2^-17 of their sizes; the weight's gradient by 2^-17 of the sum of |grad_y n| (rows of a
thread, then partial sums, some hundred additions in all)."""
import importlib

import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps      # a step of the subnormal numbers


def close(a, ref, size, slack):
    """|a - ref| within half a step of a's type and slack of `size`"""
    lim = ref.abs() * half(a.dtype) * (1 + slack) + slack * size + tiny(a.dtype)
    bad = (a.double() - ref).abs() > lim
    assert not bad.any(), (int(bad.sum()), float(((a.double() - ref).abs() - lim).max()))


def make(T, K, dt, wt=None, seed=0):
    g = gen(seed)
    x = (torch.randn(T, K, generator=g, device=DEV) * (0.3 + torch.rand(T, 1, generator=g, device=DEV))).to(dt)
    r = (torch.randn(T, K, generator=g, device=DEV) * 3).to(dt)
    w = (1 + 0.3 * torch.randn(K, generator=g, device=DEV)).to(wt or dt)
    return x, r, w


def norm64(h, w):
    h = h.double()
    rstd = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS)
    return h * rstd * w.double(), rstd


def check_codes(q, scale, y):
    K = y.shape[-1]
    blocks = torch.nn.functional.pad(y, (0, -K % 128)).unflatten(-1, (-1, 128))
    amax = blocks.abs().amax(-1).clamp(min=2.0 ** -100)
    assert scale.dtype == F32 and scale.shape == amax.shape and q.dtype == torch.float8_e4m3fn and q.shape == y.shape
    assert ((scale.double() - amax / 448).abs() <= amax / 448 * 2.0 ** -18).all()
    want = (blocks * (448 / amax)[..., None]).flatten(-2)[..., :K]
    lim = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10)) + want.abs() * 2.0 ** -17
    assert ((q.double() - want).abs() <= lim).all()


TYPES = [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (F32, F32)]


@pytest.mark.parametrize("dt,wt", TYPES)
@pytest.mark.parametrize("T,K", [(1, 1), (1, 4096), (3, 37), (5, 8), (1000, 128), (333, 1024), (300, 1025), (257, 1037), (149, 1032), (148, 2048), (700, 4096),
                                 (20, 5000), (500, 8192), (200, 8200), (3, 16384), (160, 16384), (160, 16383)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward(pkg, dt, wt, T, K, residual):
    x, r, w = make(T, K, dt, wt)
    if residual:
        y, h = pkg.rms_norm(x, w, r, EPS)
        assert torch.equal(h, (x.float() + r.float()).to(dt))
    else:
        y, h = pkg.rms_norm(x, w, eps=EPS), x
    ref, _ = norm64(h, w)
    assert y.dtype == dt
    close(y, ref, ref.abs(), 2.0 ** -19)
    if K % 8 == 0:
        for want_y in (False, True):
            out = pkg.rms_norm_fp8_block(x, w, r if residual else None, EPS, return_norm=want_y)
            check_codes(out[0], out[1], ref)
            assert len(out) == 2 + want_y + residual
            assert not want_y or torch.equal(out[2], y)
            assert not residual or torch.equal(out[-1], h)


@pytest.mark.parametrize("dt,wt", TYPES)
@pytest.mark.parametrize("T,K", [(1, 1), (1, 4096), (3, 37), (9, 8), (1000, 128), (3333, 1024), (3000, 1025), (2570, 1032), (148, 2048), (5000, 2048), (700, 4096),
                                 (301, 5000), (400, 8200), (3, 16384), (300, 16383)])
@pytest.mark.parametrize("used", ["y", "yh"])
def test_gradients(pkg, dt, wt, T, K, used):
    x, r, w = (t.requires_grad_() for t in make(T, K, dt, wt, 1))
    y, h = pkg.rms_norm(x, w, r, EPS)
    g = gen(2)
    gy, gh = (torch.randn(T, K, generator=g, device=DEV).to(dt) for _ in range(2))
    outs, gs = ([y, h], [gy, gh]) if used == "yh" else ([y], [gy])
    gx, gr, gw = torch.autograd.grad(outs, [x, r, w], gs)
    assert gx.dtype == gr.dtype == dt and gw.dtype == wt and torch.equal(gx, gr)
    n, rstd = norm64(h.detach(), torch.ones_like(w.detach()))
    d = gy.double() * w.detach().double()
    back = (d * n).mean(-1, keepdim=True)
    ref, size = rstd * (d - n * back), rstd * (d.abs() + n.abs() * (d * n).abs().mean(-1, keepdim=True))
    if used == "yh":
        ref, size = ref + gh.double(), size + gh.double().abs()
    close(gx, ref, size, 2.0 ** -17)
    close(gw, (gy.double() * n).sum(0), (gy.double() * n).abs().sum(0), 2.0 ** -17)
    again = torch.autograd.grad(pkg.rms_norm(x, w, r, EPS)[:len(outs)], [x, r, w], gs)
    assert all(torch.equal(a, b) for a, b in zip((gx, gr, gw), again))


def test_gradient_against_differences(pkg):
    """Of the kernels' own forward in fp32, along one direction of each input.  Tolerance: the forward's error 2^-19 |y| over the step, and what the
    difference quotient of the formula itself, in 64 bits, is off by."""
    T, K = 7, 300
    x, r, w = make(T, K, F32, seed=3)
    gy, gh = (torch.randn(T, K, generator=gen(4 + i), device=DEV) for i in range(2))
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    grads = torch.autograd.grad(pkg.rms_norm(leaves[0], leaves[2], leaves[1], EPS), leaves, [gy, gh])

    def own(x, r, w):
        y, h = pkg.rms_norm(x, w, r, EPS)
        return float((y.double() * gy).sum() + (h.double() * gh).sum())

    def formula(x, r, w):
        x, r = x.double(), r.double()
        return float((norm64(x + r, w.double())[0] * gy).sum() + ((x + r) * gh).sum())

    step = 2.0 ** -5
    y, h = (t.double() for t in pkg.rms_norm(x, w, r, EPS))
    for i in range(3):
        u = torch.randn((x, r, w)[i].shape, generator=gen(9 + i), device=DEV)
        ends = [[t + s * step * u if j == i else t for j, t in enumerate((x, r, w))] for s in (1, -1)]
        along = float((grads[i].double() * u).sum())
        diff, diff64 = ((f(*ends[0]) - f(*ends[1])) / (2 * step) for f in (own, formula))
        lim = (2.0 ** -18 * float((y * gy).abs().sum()) + 2.0 ** -22 * float((h * gh).abs().sum())) / step
        x64 = [t.double().requires_grad_() for t in (x, r, w)]
        n64 = norm64(x64[0] + x64[1], x64[2])[0]
        exact = float((torch.autograd.grad((n64 * gy).sum() + ((x64[0] + x64[1]) * gh).sum(), x64)[i] * u).sum())
        assert abs(along - exact) <= 2.0 ** -17 * float((grads[i].double() * u).abs().sum()) + lim
        assert abs(diff - along) <= lim + 1.1 * abs(diff64 - exact) + abs(along - exact)


@pytest.mark.parametrize("K", [1040, 136, 37])
def test_layouts(pkg, K):
    """Rows inside wider ones, off a vector's boundary, in three dimensions, transposed, broadcast.  A row off a boundary is summed in another order
    than one on it, so y need not have the same bits: each obeys the bound above, from the same h, whose bits are the same."""
    wide = torch.randn(40, 3 * K + 5, generator=gen(0), device=DEV).to(BF)
    _, r, w = make(40, K, BF)
    for x in (wide[:, :K], wide[:, K:2 * K], wide[:, 3:3 + K], wide[::2, 1:1 + K], wide[:, : 2 * K : 2], wide[0, :K].expand(40, K),
              wide[:, :K].unflatten(0, (5, 8)), wide[:, :K].unflatten(0, (5, 8)).transpose(0, 1), wide[3, :K], wide[:, :K].t().contiguous().t()):
        res = r[: x.numel() // K].view(x.shape)
        total = (x.float() + res.float()).to(BF)
        ref = norm64(total, w)[0]
        for res2 in (res, torch.cat([res, res], -1)[..., :K]):
            y, h = pkg.rms_norm(x, w, res2, EPS)
            assert y.shape == h.shape == x.shape and torch.equal(h, total)
            close(y, ref, ref.abs(), 2.0 ** -19)
        alone = norm64(x, w)[0]
        close(pkg.rms_norm(x, w, eps=EPS), alone, alone.abs(), 2.0 ** -19)
        if K % 8 == 0:
            q, s, h = pkg.rms_norm_fp8_block(x, w, res, EPS)
            assert s.shape == (*x.shape[:-1], -(-K // 128)) and torch.equal(h, total)
            check_codes(q, s, ref)
    # gradients of a view, of a broadcast row and with a broadcast gradient
    leaf = wide.clone().requires_grad_()
    w1 = w.clone().requires_grad_()
    pkg.rms_norm(leaf[:, 3:3 + K], w1, eps=EPS).float().sum().backward()
    n, rstd = norm64(wide[:, 3:3 + K], torch.ones_like(w))
    d = w.double().expand_as(n)
    back = (d * n).mean(-1, keepdim=True)
    close(leaf.grad[:, 3:3 + K], rstd * (d - n * back), rstd * (d.abs() + n.abs() * (d * n).abs().mean(-1, keepdim=True)), 2.0 ** -17)
    close(w1.grad, n.sum(0), n.abs().sum(0), 2.0 ** -17)
    assert (leaf.grad[:, 3 + K:] == 0).all() and (leaf.grad[:, :3] == 0).all()
    one = wide[0, :K].clone().requires_grad_()
    y, h = pkg.rms_norm(r[:, :K], w, one.expand(40, K), EPS)
    (y.float().square().sum() + h.float().sum()).backward()
    assert one.grad.shape == (K,) and torch.isfinite(one.grad).all()


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("T,K", [(6, 2048), (600, 2048), (600, 1037)])
@pytest.mark.parametrize("size", [1e-17, 1e15])
def test_small_and_large_rows(pkg, dt, T, K, size):
    """Without eps, rows whose squares are near the ends of fp32's range and whose gradients are as far at the other end."""
    x, _, w = make(T, K, dt, F32, 6)
    x = (x.float() * size).to(dt).requires_grad_()
    gy = torch.randn(T, K, generator=gen(8), device=DEV).to(dt)
    y = pkg.rms_norm(x, w, eps=0)
    h = x.detach().double()
    rstd = 1 / torch.sqrt(h.square().mean(-1, keepdim=True))
    n, d = h * rstd, gy.double() * w.double()
    close(y.detach(), n * w.double(), (n * w.double()).abs(), 2.0 ** -19)
    gx, = torch.autograd.grad(y, x, gy)
    back = (d * n).mean(-1, keepdim=True)
    close(gx, rstd * (d - n * back), rstd * (d.abs() + n.abs() * (d * n).abs().mean(-1, keepdim=True)), 2.0 ** -17)


def test_inference_mode(pkg):
    x, r, w = make(200, 256, BF)
    with torch.inference_mode():
        q, s, y, h = pkg.rms_norm_fp8_block(x, w, r, EPS, return_norm=True)
    want = pkg.rms_norm_fp8_block(x, w, r, EPS, return_norm=True)
    assert all(torch.equal(a.float(), b.float()) for a, b in zip((q, s, y, h), want))


def test_empty_and_unused(pkg):
    x, r, w = (t.requires_grad_() for t in make(0, 64, BF))
    y, h = pkg.rms_norm(x, w, r)
    q, s = pkg.rms_norm_fp8_block(x, w)
    assert y.shape == h.shape == q.shape == (0, 64) and s.shape == (0, 1)
    (y.sum() + h.sum()).backward()
    assert x.grad.shape == (0, 64) and (w.grad == 0).all()
    x, r, w = (t.requires_grad_() for t in make(40, 128, BF))
    q, s, h = pkg.rms_norm_fp8_block(x, w, r)
    assert not q.requires_grad and not s.requires_grad
    gx, gr, gw = torch.autograd.grad(h, [x, r, w], torch.ones_like(h), allow_unused=True)
    assert (gx == 1).all() and (gr == 1).all() and gw is None
    y, h = pkg.rms_norm(x, w.detach(), r.detach())
    assert torch.equal(torch.autograd.grad(y, x, h.detach())[0], torch.autograd.grad(pkg.rms_norm(x, w, r)[0], [x, w], h.detach())[0])
    y, _ = pkg.rms_norm(x.detach(), w, r.detach())
    assert torch.equal(torch.autograd.grad(y, w, h.detach())[0], torch.autograd.grad(pkg.rms_norm(x, w, r)[0], w, h.detach())[0])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g = torch.autograd.grad(pkg.rms_norm(x, w, r)[0].float().square().sum(), x, create_graph=True)[0]
        g.float().sum().backward()


def test_special_values(pkg):
    """A row with NaN is NaN; infinity gives what the formula gives; other rows are as without them.  Rows of zeros give zeros."""
    x, r, w = make(300, 512, BF)
    clean = [t.clone() for t in pkg.rms_norm_fp8_block(x, w, r, EPS, return_norm=True)]
    x2 = x.clone()
    x2[3, 7], x2[200, 500], x2[299] = float("nan"), float("inf"), 0
    r2 = r.clone()
    r2[299] = 0
    q, s, y, h = pkg.rms_norm_fp8_block(x2, w, r2, EPS, return_norm=True)
    keep = torch.ones(300, dtype=torch.bool, device=DEV)
    keep[[3, 200, 299]] = False
    for a, b in zip((q.float(), s, y, h), (clean[0].float(), *clean[1:])):
        assert torch.equal(a[keep], b[keep])
    assert y[3].isnan().all() and q[3].float().isnan().all() and y[200, 500].isnan() and (y[200, :500] == 0).all()
    assert (y[299] == 0).all() and (q[299].float() == 0).all() and torch.isfinite(s[299]).all()


def test_streams_and_graphs(pkg):
    x, r, w = make(600, 2048, BF)
    gy = torch.randn(600, 2048, generator=gen(5), device=DEV).to(BF)

    def step(x, r, w):
        q, s, y, h = pkg.rms_norm_fp8_block(x, w, r, EPS, return_norm=True)
        return [q.float(), s, y.detach(), h.detach(), *torch.autograd.grad([y, h], [x, r, w], [gy, gy])]

    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    want = [t.clone() for t in step(*leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step(*leaves)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = [t.clone().requires_grad_() for t in (x, r, w)]
    graphs, outs = [], []
    for _ in range(2):      # two graphs of the same tensors
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*static))
    with torch.no_grad():
        for t, seed in zip(static, (11, 12, 13)):
            t.copy_(torch.randn(t.shape, generator=gen(seed), device=DEV).to(BF))
    for g in graphs:
        g.replay()
    want = step(*static)
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traced_and_forward_gradients(pkg):
    x, r, w = make(40, 256, BF)
    for fn in (lambda x, r: pkg.rms_norm(x, w, r, EPS), lambda x, r: [t.float() for t in pkg.rms_norm_fp8_block(x, w, r, EPS, return_norm=True)]):
        with torch.no_grad():
            traced = torch.jit.trace(fn, (x, r))
            for n in (40, 7, 300):
                a, b = (t.float().mean(0, keepdim=True).expand(n, -1).contiguous().to(BF) for t in (x, r))
                assert all(torch.equal(p, q) for p, q in zip(traced(a, b), fn(a, b)))
        with fw.dual_level(), pytest.raises(Exception, match="forward"):
            fn(fw.make_dual(x, torch.ones_like(x)), r)


def test_observer(pkg):
    x, r, w = (t.requires_grad_() for t in make(300, 256, BF))
    names = []
    pkg.ops.set_hook(lambda name, launches, a, b: names.append((name, launches)))
    try:
        pkg.rms_norm(x, w, r)[0].sum().backward()
    finally:
        pkg.ops.set_hook(None)
    torch.cuda.synchronize()
    assert names == [("rms_norm_fwd", 1), ("rms_norm_bwd", 2)]


# ------------------------------------------------------------------------------------------------ products of rows that are codes already
@pytest.mark.parametrize("M", [0, 1, 4, 16, 17, 64, 300, 3001])
@pytest.mark.parametrize("N,K", [(680, 1040), (4096, 2048), (64, 64), (512, 272)])
def test_product_of_codes(pkg, M, N, K):
    """The same bits as quantised on the way, from the scales of the quantiser (copied) and at the norm's pitch (read in place)."""
    g = gen(M)
    x = torch.randn(M, K, generator=g, device=DEV).to(BF)
    w, s = pkg.fp8_block_quantize_weight(torch.randn(N, K, generator=g, device=DEV).to(BF))
    want = pkg.fp8_block_linear(x, w, s)
    q, qs = pkg.fp8_block_quantize(x)
    assert torch.equal(pkg.fp8_block_linear(None, w, s, quantized=(q, qs)), want)
    assert torch.equal(pkg.fp8_block_linear(x, w, s, (q, qs.contiguous())), want)
    room = torch.full((qs.shape[1], -(-M // 128) * 128 + 128), float("nan"), device=DEV)
    room[:, :M] = qs.t()
    assert torch.equal(pkg.fp8_block_linear(x, w, s, quantized=(q, room[:, :M].t())), want)
    if M and M % 2 == 0:
        assert torch.equal(pkg.fp8_block_linear(None, w, s, quantized=(q.view(2, -1, K), qs.reshape(2, M // 2, -1))), want.view(2, -1, N))
    pkg.check_status()


def test_norm_into_product(pkg):
    """Norm, then the product of its codes: against 64 bits on those codes, and the gradient that goes through y."""
    T, K, N = 500, 1040, 680
    x, r, wn = (t.requires_grad_() for t in make(T, K, BF))
    w, s = pkg.fp8_block_quantize_weight((torch.randn(N, K, generator=gen(7), device=DEV) * 0.05).to(BF))
    q, qs, y, h = pkg.rms_norm_fp8_block(x, wn, r, EPS, return_norm=True)
    out = pkg.fp8_block_linear(y, w, s, quantized=(q, qs))
    pad = lambda sc, n: sc.double().repeat_interleave(128, -1)[..., :n]      # noqa: E731
    w64 = w.double() * pad(s, K).repeat_interleave(128, 0)[:N]
    x64 = q.double() * pad(qs, K)
    # fp32 sums of K products, each block's scaled: K 2^-24 of the products' sizes, and half a step
    close(out.detach(), x64 @ w64.t(), x64.abs() @ w64.abs().t(), K * 2.0 ** -24)
    go = torch.randn(T, N, generator=gen(8), device=DEV).to(BF)
    got = torch.autograd.grad([out, h], [x, r, wn], [go, torch.ones_like(h)], retain_graph=True)
    y2 = y.detach().requires_grad_()
    gy = torch.autograd.grad(pkg.fp8_block_linear(y2, w, s), y2, go)[0]
    want = torch.autograd.grad(pkg.rms_norm(x, wn, r, EPS), [x, r, wn], [gy, torch.ones_like(h)])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pkg.check_status()


@pytest.mark.parametrize("compiled", [True, False])
def test_compiled_and_python_functions_agree(pkg, monkeypatch, compiled):
    if not compiled:
        monkeypatch.setattr(importlib.import_module(pkg.__name__ + "._lib"), "fast", lambda: None)
    x, r, w = (t.requires_grad_() for t in make(200, 520, BF))
    q, s, y, h = pkg.rms_norm_fp8_block(x, w, r, EPS, return_norm=True)
    ref, _ = norm64(h.detach(), w.detach())
    close(y.detach(), ref, ref.abs(), 2.0 ** -19)
    check_codes(q, s, ref)
    assert y.requires_grad and h.requires_grad and not q.requires_grad
    gx, gr = torch.autograd.grad([y, h], [x, r], [torch.ones_like(y), torch.ones_like(y)])
    assert torch.equal(gx, gr)


def test_refusals(pkg):
    x, r, w = make(4, 128, BF)
    wq, ws = pkg.fp8_block_quantize_weight(torch.ones(64, 128, dtype=BF, device=DEV))
    q, s = pkg.fp8_block_quantize(x)
    for match, call in (("multiple of 8", lambda: pkg.rms_norm_fp8_block(x[:, :100], w[:100])),
                        ("weight must be", lambda: pkg.rms_norm(x, w[:64])), ("weight must be", lambda: pkg.rms_norm(x, w.half())),
                        ("bfloat16, float16 or float32", lambda: pkg.rms_norm(x.double(), w)), ("residual", lambda: pkg.rms_norm(x, w, r[:2])),
                        ("residual", lambda: pkg.rms_norm(x, w, r.float())), ("eps", lambda: pkg.rms_norm(x, w, eps=-1.0)),
                        ("last dimension", lambda: pkg.rms_norm(x[:, :0], w[:0])), ("codes must be", lambda: pkg.fp8_block_linear(x, wq, ws, (x, s))),
                        ("scales must be", lambda: pkg.fp8_block_linear(x, wq, ws, (q, s[:2]))), ("codes' shape", lambda: pkg.fp8_block_linear(x[:2], wq, ws, (q, s))),
                        ("take no gradient", lambda: pkg.fp8_block_linear(x, wq, ws, (q, s.clone().requires_grad_())))):
        with pytest.raises(ValueError, match=match):
            call()


def test_an_infinite_eps_is_refused(pkg):
    x, _, w = make(4, 128, BF)
    for eps in (float("inf"), 1e39, float("nan")):
        for call in (lambda: pkg.rms_norm(x, w, eps=eps), lambda: pkg.rms_norm(x[:, ::2], w[::2], eps=eps), lambda: pkg.rms_norm_fp8_block(x, w, eps=eps)):
            with pytest.raises(ValueError, match="eps"):
                call()


def test_offsets_beyond_32_bits(pkg):
    """More than 2^31 values; rows do not depend on where they lie."""
    T, K, m = 135_000, 16_384, 1000
    g = torch.Generator(device=DEV).manual_seed(41)
    x, r = (torch.empty(T, K, dtype=BF, device=DEV).normal_(generator=g) for _ in range(2))
    w = torch.empty(K, dtype=BF, device=DEV).normal_(generator=g)
    few = [t[-m:].clone() for t in (x, r)]
    q, s, y, h = pkg.rms_norm_fp8_block(x, w, r, return_norm=True)
    for got, want in zip((q, s, y, h), pkg.rms_norm_fp8_block(few[0], w, few[1], return_norm=True)):
        assert torch.equal(got[-m:].float(), want.float())
    del q, s, y, h
    gy = torch.zeros(T, K, dtype=BF, device=DEV)
    gy[-m:].normal_(generator=g)
    out = []
    for rows in ((x, r, gy), (few[0], few[1], gy[-m:])):
        p, res, go = rows[0].detach().requires_grad_(), rows[1], rows[2]
        wl = w.detach().requires_grad_()
        y, h = pkg.rms_norm(p, wl, res)
        gx, gw = torch.autograd.grad([y, h], [p, wl], [go, go])
        out.append((gx[-m:].clone(), gw.float()))
        del y, h, gx
    assert torch.equal(out[0][0], out[1][0])
    assert float((out[0][1] - out[1][1]).norm()) <= 2.0 ** -7 * float(out[1][1].norm())      # each rounded to bf16 once, sums in another order
    pkg.check_status()
