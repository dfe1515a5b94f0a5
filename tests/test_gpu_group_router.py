"""GPU: group-limited top-k (`group_topk`, `fused_group_router`) against a 64-bit restatement: picks equal everywhere, weights and
gradients within bounds counted in roundings.

Steps of 2^-23 (fp32).  A sigmoid: exponential 2, sum 0.5, quotient 1; its weight: sum of k 2.5, quotient 1, scale 0.5: below 8 = 2^-20.
A softmax whose logits span D: exponential 2, the denominator's exponentials 2 + 1.17 D, its sum 6.5, quotient and product 2, the weight 4:
for D <= 9 below 32 = 2^-18.  A gradient is a difference of terms up to |g| / t, each with such an error and twice as many
operations: 2^-17 of that, and one rounding to the logits' type."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def scores64(z, scoring):
    z = z.double()
    if scoring == "sigmoid":
        return torch.sigmoid(z)
    return torch.where((z == -torch.inf).all(1, keepdim=True), torch.zeros_like(z), torch.softmax(z, 1))


def route64(z, k, bias=None, groups=1, opened=None, scoring="sigmoid", by="top2", norm=True, scale=1.0):
    """(idx, weights) of logits (N,E); equal values in the order of the experts, decided by the logits where they decide."""
    opened = groups if opened is None else opened
    s = scores64(z, scoring)
    v = s if bias is None else s + bias.double()
    order = z.double() if bias is None else v
    N, E = z.shape
    if opened < groups:
        x = (order if by == "max" else v).view(N, groups, E // groups)
        top = x.sort(dim=2, descending=True).values
        value = top[..., 0] if by == "max" or E == groups else top[..., 0] + top[..., 1]
        keep = torch.zeros(N, groups, dtype=torch.bool, device=z.device)
        keep.scatter_(1, value.sort(dim=1, descending=True, stable=True).indices[:, :opened], True)
        # closed experts behind every open one, also behind open ones of -inf
        closed = ~keep.repeat_interleave(E // groups, 1)
        first = order.sort(dim=1, descending=True, stable=True).indices
        idx = first.gather(1, closed.gather(1, first).long().sort(dim=1, stable=True).indices)[:, :k]
    else:
        idx = order.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, idx)
    if norm and k > 1:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return idx, w * scale


def grad64(z, idx, g, scoring, norm, scale):
    s = scores64(z, scoring)
    raw, g = s.gather(1, idx), g.double() * scale
    if norm and idx.shape[1] > 1:
        t = raw.sum(1, keepdim=True) + 1e-20
        g = (g - (g * raw).sum(1, keepdim=True) / t) / t
    ds = torch.zeros_like(s).scatter(1, idx, g)
    if scoring == "sigmoid":
        return ds * s * torch.sigmoid(-z.double())
    return s * (ds - (ds * s).sum(1, keepdim=True))


def make(T, E, dtype, seed, bias):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = (torch.randn(T, E, generator=g, device=DEV) * 1.5).clamp(-4.5, 4.5).to(dtype)
    b = (torch.randn(E, generator=g, device=DEV) * 0.1) if bias else None
    return z, b, g


CASES = [   # T, E, k, groups, open
    (1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (2, 8, 8, 1, 1), (3, 8, 2, 8, 3), (5, 60, 4, 4, 2), (7, 255, 5, 3, 1), (33, 96, 6, 6, 5), (40, 252, 14, 9, 2),
    (64, 256, 32, 1, 1), (65, 17, 3, 17, 6), (129, 64, 6, 1, 1), (130, 128, 8, 16, 16), (31, 256, 32, 32, 4), (4000, 160, 6, 8, 3), (20011, 256, 8, 8, 4),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,bias,by", list(itertools.product(("sigmoid", "softmax"), (False, True), ("top2", "max"))))
def test_picks_weights_counts_and_gradient(pkg, dtype, scoring, bias, by):
    for n, (T, E, k, groups, opened) in enumerate(CASES):
        norm, scale = n % 3 != 0, 1.0 if n % 2 else 2.5
        z, b, g = make(T, E, dtype, n, bias)
        z.requires_grad_(True)
        idx, w, counts = pkg.group_topk(z, k, b, groups, opened, scoring, by, norm, scale, return_counts=True)
        ri, rw = route64(z.detach(), k, b, groups, opened, scoring, by, norm, scale)
        assert torch.equal(idx, ri), (T, E, k, groups, opened, int((idx != ri).any(1).sum()))
        assert torch.equal(counts.long(), torch.bincount(ri.reshape(-1), minlength=E))
        steps = 2.0 ** (-20 if scoring == "sigmoid" else -18)
        assert ((w - rw).abs() <= steps * rw).all(), (T, E, float(((w - rw).abs() / rw).max()))
        gw = torch.randn(T, k, generator=g, device=DEV)
        (got,) = torch.autograd.grad(w, z, gw)
        ref = grad64(z.detach(), ri, gw, scoring, norm, scale)
        assert got.dtype == dtype
        t = rw.sum(1, keepdim=True) / scale if not norm or k == 1 else torch.ones_like(rw[:, :1])
        s = scores64(z.detach(), scoring).gather(1, ri).sum(1, keepdim=True)
        size = 2 * scale * gw.abs().double().max(1, keepdim=True).values / (s if norm and k > 1 else t.clamp(min=1.0))
        bound = 2.0 ** -17 * size * scores64(z.detach(), scoring) + torch.finfo(dtype).eps / 2 * ref.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert ((got.double() - ref).abs() <= bound).all(), (T, E, k, scoring, norm, float(((got.double() - ref).abs() / bound).max()))


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_gradient_is_what_differences_give(pkg, scoring):
    """Along a direction d: (w(z + h d) - w(z - h d)) / 2h, h = 2^-7.  The third derivative of a weight along a unit direction is below 2
    (shares of shares of at most 1), so the formula is off by h^2 / 6 * 2 = 2e-5 at most; the two weights by 2^-18 each over 2h: 2.5e-4; sums of
    k = 4 weights with |g| <= 1: four times that."""
    E, k, h = 32, 4, 2.0 ** -7
    z = torch.linspace(-2.0, 2.0, E, device=DEV)[torch.randperm(E, generator=torch.Generator().manual_seed(0)).to(DEV)].repeat(64, 1).contiguous()
    gen = torch.Generator(device=DEV).manual_seed(1)
    d = torch.nn.functional.normalize(torch.randn(64, E, generator=gen, device=DEV), dim=1)
    g = torch.rand(64, k, generator=gen, device=DEV) * 2 - 1
    z.requires_grad_(True)
    idx, w = pkg.group_topk(z, k, scoring=scoring)
    (dz,) = torch.autograd.grad(w, z, g)
    up, dn = (pkg.group_topk((z + s * h * d).detach(), k, scoring=scoring) for s in (1, -1))
    assert torch.equal(up[0].sort(1).values, idx.sort(1).values) and torch.equal(dn[0].sort(1).values, idx.sort(1).values)
    by = lambda r: torch.zeros(64, E, device=DEV).scatter(1, *r).gather(1, idx)    # noqa: E731  in the order of the picks at z
    num = ((by(up) - by(dn)).double() / (2 * h) * g).sum(1)
    assert ((dz * d).double().sum(1) - num).abs().max() <= 4 * (2e-5 + 2.5e-4)


def test_values_that_fp32_does_not_tell_apart(pkg):
    """Pairs of experts whose score plus bias differ by less than a rounding of fp32: the pick is that of 64 bits, in both directions."""
    T, E = 4096, 64
    g = torch.Generator(device=DEV).manual_seed(5)
    for scoring in ("sigmoid", "softmax"):
        z = (torch.randn(T, E, generator=g, device=DEV)).clamp(-3, 3)
        b = torch.zeros(E, device=DEV)
        s = scores64(z[:1], scoring)[0]
        b[1::2] = (s[0::2] - s[1::2]).float()          # expert 2i+1 level with 2i, to the last bit of the bias
        z = z[:1].expand(T, E).contiguous()
        z[1:, 2:] += torch.randn(T - 1, E - 2, generator=g, device=DEV) * (1e-6 if scoring == "sigmoid" else 0.0)
        for groups, opened in ((1, 1), (8, 4), (32, 5)):
            k = 6
            idx, w = pkg.group_topk(z, k, b, groups, opened, scoring, "max")
            ri, rw = route64(z, k, b, groups, opened, scoring, "max")
            assert torch.equal(idx, ri), (scoring, groups, int((idx != ri).any(1).sum()))


@pytest.mark.parametrize("scoring,bias", list(itertools.product(("sigmoid", "softmax"), (False, True))))
def test_equal_logits_infinities_and_nan(pkg, scoring, bias):
    E, k = 256, 8
    z = torch.zeros(12, E, device=DEV)
    b = torch.zeros(E, device=DEV) if bias else None
    z[1] = -torch.inf
    z[2, 5:] = -torch.inf                      # fewer experts than picks
    z[3, 7] = torch.inf
    z[4] = 60.0                                # sigmoid is 1 in fp32
    z[4, 100:110] = torch.arange(60.0, 70.0)
    z[5] = -200.0
    z[6] = torch.arange(E) % 5                 # 51 equal best ones
    z[7, ::3] = -0.0
    for groups, opened in ((1, 1), (8, 2), (8, 8)):
        zz = z.clone()
        if scoring == "softmax":
            zz[3, 7] = 50.0
        zz.requires_grad_(True)
        idx, w, counts = pkg.group_topk(zz, k, b, groups, opened, scoring, "max", return_counts=True)
        ri, rw = route64(zz.detach(), k, b, groups, opened, scoring, "max")
        rows = [r for r in range(12) if not (bias and r == 4)]       # score + bias of row 4 is equal in 64 bits too where scores are 1
        assert torch.equal(idx[rows], ri[rows]), (groups, opened, (idx != ri).any(1).nonzero().flatten().tolist())
        assert int(counts.sum()) == 12 * k and (idx.sort(1).values.diff(dim=1) > 0).all()
        assert torch.isfinite(w).all() and ((w[rows] - rw[rows]).abs() <= 2.0 ** -18 * rw[rows] + 1e-12).all()
        (g,) = torch.autograd.grad(w, zz, torch.ones_like(w))
        assert torch.isfinite(g).all() and (g[1] == 0).all()
    z[9, 40] = torch.nan
    idx, w = pkg.group_topk(z, k, b, scoring=scoring)
    if scoring == "sigmoid":
        assert int(idx[9, 0]) == 40 and (idx[9].sort().values.diff() > 0).all()
    else:                                      # the whole row's scores are NaN
        assert (idx[9].sort().values.diff() > 0).all()
    assert torch.isnan(w[9, 0]) and torch.isfinite(w[8]).all() and torch.isfinite(w[10]).all()


@pytest.mark.parametrize("E,k,groups,opened", [(8, 3, 1, 1), (24, 4, 1, 1), (24, 4, 4, 2), (64, 6, 8, 3), (256, 8, 8, 4)])
@pytest.mark.parametrize("scoring", ("sigmoid", "softmax"))
def test_scores_and_biases_that_are_not_finite(pkg, scoring, E, k, groups, opened):
    """Infinite biases open and close experts; NaN, of a bias or of a softmax over +infinity, ranks first and counts as infinity in a group."""
    z, b, _ = make(70, E, torch.float32, 5, True)

    def check(z, b):
        v = scores64(z, scoring) + b.double()
        for by in ("top2", "max"):
            idx, w, counts = pkg.group_topk(z, k, b, groups, opened, scoring, by, return_counts=True)
            if opened < groups:
                top = v.nan_to_num(nan=torch.inf, posinf=torch.inf, neginf=-torch.inf).view(-1, groups, E // groups).sort(dim=2, descending=True).values
                value = top[..., 0] if by == "max" else (top[..., 0] + top[..., 1]).nan_to_num(nan=torch.inf, posinf=torch.inf, neginf=-torch.inf)
                keep = torch.zeros(z.shape[0], groups, dtype=torch.bool, device=DEV)
                keep.scatter_(1, value.sort(dim=1, descending=True, stable=True).indices[:, :opened], True)
                open_ = keep.repeat_interleave(E // groups, 1)
            else:
                open_ = torch.ones_like(v, dtype=torch.bool)
            # NaN first, then by value, in the order of the experts; closed ones last
            order = v.nan_to_num(nan=0.0, posinf=torch.inf, neginf=-torch.inf).sort(dim=1, descending=True, stable=True).indices
            for first in (v.isnan(), open_):
                rank = (~first).gather(1, order).long().sort(dim=1, stable=True).indices
                order = order.gather(1, rank)
            assert torch.equal(idx, order[:, :k]), (by, (idx != order[:, :k]).any(1).nonzero().flatten().tolist()[:5])
            assert int(counts.sum()) == z.shape[0] * k
            s = scores64(z, scoring).gather(1, idx)
            s = s / (s.sum(1, keepdim=True) + 1e-20)
            assert torch.equal(w.isnan(), s.isnan())
            assert ((w - s).abs() <= 2.0 ** -18 * s)[~s.isnan()].all()

    closed = b.clone()
    closed[::3] = -torch.inf
    check(z, closed)
    both = closed.clone()
    both[E // 2 + 1] = torch.inf
    check(z, both)
    if groups > 1:                             # one group has nothing but +infinity and -infinity
        both[-(E // groups):] = -torch.inf
        both[-1] = torch.inf
        check(z, both)
    nan = b.clone()
    nan[E - 2] = torch.nan
    check(z, nan)
    if scoring == "softmax":
        z = z.clone()
        z[::2, 5] = torch.inf
        check(z, b)


def test_empty_strided_unaligned_and_three_dimensional(pkg):
    z, b, _ = make(400, 64, torch.bfloat16, 3, True)
    ref = pkg.group_topk(z, 6, b, 8, 3, return_counts=True)
    idx, w, c = pkg.group_topk(z[:0], 6, b, 8, 3, return_counts=True)
    assert idx.shape == (0, 6) and w.shape == (0, 6) and int(c.sum()) == 0
    wide = torch.empty(400, 100, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:67] = z
    for got in (pkg.group_topk(wide[:, 3:67], 6, b, 8, 3, return_counts=True),
                pkg.group_topk(z.view(8, 50, 64), 6, b.double(), 8, 3, return_counts=True)):
        assert torch.equal(got[0].reshape(400, 6), ref[0]) and torch.equal(got[1].reshape(400, 6), ref[1]) and torch.equal(got[2], ref[2])
    odd = torch.empty(400 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(400, 64)      # two bytes past a boundary
    odd.copy_(z)
    odd.requires_grad_(True)
    got = pkg.group_topk(odd, 6, b, 8, 3)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    (go,) = torch.autograd.grad(got[1].sum(), odd)
    z.requires_grad_(True)
    (gz,) = torch.autograd.grad(pkg.group_topk(z, 6, b, 8, 3)[1].sum(), z)
    assert torch.equal(go, gz)


def test_offsets_past_32_bits(pkg):
    T, E = (1 << 23) + 9, 256      # 2^31 + 2304 logits
    z = torch.zeros(T, E, dtype=torch.bfloat16, device=DEV)
    tail, b, _ = make(64, E, torch.bfloat16, 9, True)
    z[-64:] = tail
    z[:-64, 3] = 1.0
    z.requires_grad_(True)
    idx, w = pkg.group_topk(z, 1, None, 1, 1, "sigmoid")
    ri, rw = route64(tail, 1)
    assert torch.equal(idx[-64:], ri) and (idx[:-64] == 3).all()
    (g,) = torch.autograd.grad(w, z, torch.ones_like(w))
    ref = grad64(tail, ri, torch.ones(64, 1, device=DEV), "sigmoid", True, 1.0)
    assert ((g[-64:].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -17).all()


def test_another_stream_and_a_captured_graph(pkg):
    z, b, _ = make(3000, 256, torch.bfloat16, 11, True)
    ref = pkg.group_topk(z, 8, b, 8, 4, return_counts=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.group_topk(z, 8, b, 8, 4, return_counts=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, ref))
    static = torch.zeros_like(z).requires_grad_(True)
    gw = torch.ones(3000, 8, device=DEV)
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(pkg.group_topk(static, 8, b, 8, 4)[1], static, gw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.group_topk(static, 8, b, 8, 4, return_counts=True)
        (grad,) = torch.autograd.grad(out[1], static, gw)
    with torch.no_grad():
        static.copy_(z)
    for _ in range(2):
        graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, ref))
    z.requires_grad_(True)
    assert torch.equal(grad, torch.autograd.grad(pkg.group_topk(z, 8, b, 8, 4)[1], z, gw)[0])


def test_router_from_hidden_states(pkg):
    """Logits, picks and gradients of x and of the gate weight; one group and sigmoid scores are the plain router's case."""
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(4, 100, 256, generator=g, device=DEV).to(torch.bfloat16).requires_grad_(True)
    W = (torch.randn(64, 256, generator=g, device=DEV) * 0.06).to(torch.bfloat16).requires_grad_(True)
    idx, w, counts, logits = pkg.fused_group_router(x, W, None, 6, 64, 8, 3, "softmax", "max", return_counts=True, return_logits=True)
    assert idx.shape == (4, 100, 6) and logits.shape == (4, 100, 64) and int(counts.sum()) == 2400
    # 256 products of bf16 values summed in fp32, one rounding to bf16
    ref = x.detach().double().view(-1, 256) @ W.detach().double().t()
    assert ((logits.detach().double().view(-1, 64) - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -14).all()
    ri, _ = route64(logits.detach().view(-1, 64), 6, None, 8, 3, "softmax", "max")
    assert torch.equal(idx.view(-1, 6), ri)
    gw = torch.randn(4, 100, 6, generator=g, device=DEV)
    gx, gW = torch.autograd.grad(w, (x, W), gw)
    dl = grad64(logits.detach().view(-1, 64), ri, gw.view(-1, 6), "softmax", True, 1.0)
    # dl is rounded to bf16 (2^-8 of each), the product again: against the norms of what is summed
    rx, rW = dl @ W.detach().double(), dl.t() @ x.detach().double().view(-1, 256)
    bx = 2.0 ** -7 * (dl.abs() @ W.detach().double().abs()) + 2.0 ** -8 * rx.abs() + 1e-6
    bW = 2.0 ** -7 * (dl.abs().t() @ x.detach().double().view(-1, 256).abs()) + 2.0 ** -8 * rW.abs() + 1e-6
    assert ((gx.double().view(-1, 256) - rx).abs() <= bx).all() and ((gW.double() - rW).abs() <= bW).all()
    b = torch.randn(64, generator=g, device=DEV) * 0.05
    plain, group = pkg.fused_mlp_router(x, W, b, 6, 64), pkg.fused_group_router(x, W, b, 6, 64)
    same = (plain[0] == group[0]).all(-1)
    assert same.float().mean() > 0.999 and torch.allclose(plain[1][same], group[1][same], rtol=2.0 ** -19, atol=0)
    e = pkg.fused_group_router(x[:, :0], W, None, 6, 64)
    assert e[0].shape == (4, 0, 6)
