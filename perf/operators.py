"""Measurable cases of four operators of the package: group-limited routing, the routers' losses, a dense product in 8-bit
floating point with a scale per block of 128, and the experts over such weights.

`listed()` names twelve cases, `draw(rng)` gives others of the same ranges, `prepare` makes what a program holds before the call,
`run` is one pass (the package's entry points where `own` is true, elementary torch operations otherwise), `exact` the same in 64
bits, `work` the bytes and operations a pass cannot do without."""
import importlib
import math

import torch

own = False


def listed():
    return [
        # serving, the next token of one sequence: 256 experts in 8 groups of which 4 are open, fp32 logits, selection bias
        dict(name="route_decode_1", op="route", T=1, E=256, k=8, groups=8, open=4, scoring="sigmoid", bias=True, by="top2", norm=True,
             dtype="f32", pad=False, grad=False),
        # training, the same router over a large step, forward and backward; the batch ends in padding (rows of zeros)
        dict(name="route_train_32768", op="route", T=32768, E=256, k=8, groups=8, open=4, scoring="sigmoid", bias=True, by="top2", norm=True,
             dtype="bf16", pad=True, grad=True),
        # training, softmax scores without a bias: groups by their best expert, weights not renormalised, odd sizes
        dict(name="route_softmax_5003", op="route", T=5003, E=60, k=4, groups=4, open=2, scoring="softmax", bias=False, by="max", norm=False,
             dtype="f32", pad=False, grad=True),
        # the toy training step: balance and z loss of 512 tokens over 8 experts, latency and launches
        dict(name="losses_512", op="losses", B=1, S=512, E=8, k=2, scoring="softmax", per_sequence=False, mask=False, dtype="bf16"),
        # a padded batch, the balance taken sequence by sequence over normalised sigmoid scores; one slot of the batch is empty
        dict(name="losses_padded", op="losses", B=16, S=1023, E=64, k=6, scoring="sigmoid", per_sequence=True, mask=True, dtype="f32"),
        # a large training step over many experts
        dict(name="losses_32768", op="losses", B=1, S=32768, E=256, k=8, scoring="softmax", per_sequence=False, mask=False, dtype="bf16"),
        # serving, a few sequences decoding: the weights are read once
        dict(name="linear_decode_4", op="linear", T=4, N=4096, K=4096, grad=False),
        # fine-tuning beside frozen 8-bit weights, forward and gradient of the input: widths that fill no block of 128
        dict(name="linear_ragged_3001", op="linear", T=3001, N=680, K=1040, grad=True),
        # the same at the size of a large dense block
        dict(name="linear_8192", op="linear", T=8192, N=14336, K=4096, grad=True),
        # serving, one sequence through 64 experts: six of them are read
        dict(name="experts_decode_1", op="experts", T=1, E=64, H=2048, I=1408, k=6),
        # serving, a batch decoding through 8 large experts: every expert's weights are read for a few rows each
        dict(name="experts_decode_64", op="experts", T=64, E=8, H=4096, I=14336, k=2),
        # serving, prompts of a whole batch
        dict(name="experts_prefill_16384", op="experts", T=16384, E=64, H=2048, I=1408, k=6),
    ]


def _log(rng, lo, hi, mult=1):
    """A multiple of `mult` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi // mult * mult, max(-(-lo // mult) * mult, round(v / mult) * mult)))


def draw(rng):
    op = rng.choice(["route", "route", "losses", "linear", "linear", "experts", "experts"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 3, 4, 6, 8, 16])
        E = groups * rng.randint(max(1, -(-4 // groups)), 256 // groups)
        opened = rng.randint(1, groups)
        return dict(op=op, T=_log(rng, 1, 32768), E=E, k=rng.randint(1, min(16, opened * (E // groups))), groups=groups, open=opened,
                    scoring=rng.choice(["sigmoid", "softmax"]), bias=rng.random() < 0.5, by=rng.choice(["top2", "max"]),
                    norm=rng.random() < 0.7, dtype=rng.choice(["bf16", "f16", "f32"]), pad=rng.random() < 0.3, grad=rng.random() < 0.6)
    if op == "losses":
        B, E = rng.randint(1, 16), rng.randint(2, 256)
        return dict(op=op, B=B, S=_log(rng, 1, 32768 // B), E=E, k=rng.randint(1, min(8, E)), scoring=rng.choice(["sigmoid", "softmax"]),
                    per_sequence=rng.random() < 0.5, mask=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "linear":
        return dict(op=op, T=_log(rng, 1, 8192), N=_log(rng, 64, 4096, 8), K=_log(rng, 64, 4096, 16), grad=rng.random() < 0.5)
    E = rng.choice([1, 4, 8, 16, 32, 64, 128])
    return dict(op=op, T=_log(rng, 1, 8192), E=E, H=_log(rng, 256, 2048, 128), I=_log(rng, 128, 1408, 128), k=rng.randint(1, min(8, E)))


_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ inputs
def _blocks(w, kind):
    """Weights as a checkpoint holds them: (codes e4m3, a scale per block of 128 x 128), of (..., N, K)."""
    N, K = w.shape[-2:]
    nb, kb = -(-N // 128), -(-K // 128)
    p = torch.nn.functional.pad(w.float(), (0, kb * 128 - K, 0, nb * 128 - N)).unflatten(-1, (kb, 128)).unflatten(-3, (nb, 128))
    amax = p.abs().amax(dim=(-3, -1)).clamp(min=2.0 ** -100)
    codes = torch.div(p * 448.0, amax[..., :, None, :, None]).clamp(-448.0, 448.0).to(kind)
    return codes.flatten(-4, -3).flatten(-2, -1)[..., :N, :K].contiguous(), torch.div(amax, torch.full_like(amax, 448.0))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")     # noqa: E731
    c = dict(case)
    if c["op"] == "route":
        logits = rand(c["T"], c["E"]).to(_TYPES[c["dtype"]])
        if c["pad"]:
            logits[c["T"] - c["T"] // 16:] = 0
        c["logits"] = logits.requires_grad_(c["grad"])
        # a bias as its update leaves it: multiples of the update's step
        c["b"] = (rand(c["E"]) * 20).round() * 1e-3 if c["bias"] else None
        c["gw"] = rand(c["T"], c["k"])
    elif c["op"] == "losses":
        logits = (rand(c["B"], c["S"], c["E"]) * 1.5).to(_TYPES[c["dtype"]])
        c["idx"] = torch.topk(logits.float() + 0.1 * rand(c["B"], c["S"], c["E"]), c["k"], dim=-1).indices
        c["logits"] = logits.requires_grad_(True)
        c["m"] = None
        if c["mask"]:
            lengths = (torch.rand(c["B"], 1, generator=g, device="cuda") * (c["S"] + 1)).long()
            lengths[0], lengths[-1] = 0, c["S"]
            c["m"] = torch.arange(c["S"], device="cuda")[None, :] < lengths
        c["grads"] = [torch.tensor(0.01, device="cuda"), torch.tensor(0.001, device="cuda")]
    elif c["op"] == "linear":
        c["x"] = (rand(c["T"], c["K"]) * (0.5 + rand(c["T"], 1).abs())).to(torch.bfloat16).requires_grad_(c["grad"])
        c["w"], c["ws"] = _blocks(rand(c["N"], c["K"]) * 0.02 * (0.5 + rand(c["N"], 1).abs()), torch.float8_e4m3fn)
        c["gy"] = rand(c["T"], c["N"]).to(torch.bfloat16)
    else:
        T, E, H, I, k = (c[n] for n in ("T", "E", "H", "I", "k"))
        c["x"] = rand(T, H).to(torch.bfloat16)
        scores = rand(T, E)
        c["idx"] = torch.topk(scores, k, dim=-1).indices
        w = torch.sigmoid(torch.gather(scores, 1, c["idx"]))
        c["weights"] = w / w.sum(1, keepdim=True)
        stacks = [_blocks(torch.randn(n, m, generator=g, device="cuda") * 0.02, torch.float8_e4m3fn)
                  for _ in range(E) for n, m in ((2 * I, H), (H, I))]
        c["gate_up"], c["gate_up_scale"] = (torch.stack(t) for t in zip(*stacks[0::2]))
        c["down"], c["down_scale"] = (torch.stack(t) for t in zip(*stacks[1::2]))
    return c


# ------------------------------------------------------------------------------------------------ one pass
def run(c):
    return {"route": _route, "losses": _losses, "linear": _linear, "experts": _experts}[c["op"]](c)


def _pkg():
    return importlib.import_module("triton-kernel-fused_b200")


def _picks(z, c):
    """idx (T,k): the best experts of the open groups, in 64 bits, since picks are decided between values close to one another;
    equal values go to the lowest index."""
    E, G = c["E"], c["groups"]
    s = _scores(z.double(), c["scoring"])
    v = s if c["b"] is None else s + c["b"].double()
    if G > 1:
        best = v.unflatten(1, (G, E // G)).sort(dim=2, descending=True).values
        of_group = best[:, :, 0] if c["by"] == "max" or E == G else best[:, :, 0] + best[:, :, 1]
        groups = of_group.sort(dim=1, descending=True, stable=True).indices[:, :c["open"]]
        opened = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, groups, True)
        v = v.masked_fill(~opened.repeat_interleave(E // G, dim=1), -math.inf)
    return v.sort(dim=1, descending=True, stable=True).indices[:, :c["k"]]


def _scores(z, scoring):
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    e = torch.exp(z - z.amax(dim=1, keepdim=True))
    return e / e.sum(dim=1, keepdim=True)


def _route(c):
    norm = c["norm"] and c["k"] > 1
    if own:
        idx, w, counts = _pkg().group_topk(c["logits"], c["k"], bias=c["b"], num_groups=c["groups"], topk_groups=c["open"],
                                           scoring=c["scoring"], group_score=c["by"], norm_topk_prob=c["norm"],
                                           routed_scaling_factor=2.5, return_counts=True)
        if not c["grad"]:
            return {"idx": idx, "weights": w, "counts": counts}
        return {"idx": idx, "weights": w.detach(), "counts": counts, "grad": torch.autograd.grad(w, c["logits"], c["gw"])[0]}
    z = c["logits"].detach().float().requires_grad_(c["grad"])
    idx = _picks(z.detach(), c)
    raw = torch.gather(_scores(z, c["scoring"]), 1, idx)
    w = raw / (raw.sum(dim=1, keepdim=True) + 1e-20) * 2.5 if norm else raw * 2.5
    counts = torch.zeros(c["E"], dtype=torch.int32, device=z.device)
    counts.scatter_add_(0, idx.reshape(-1), torch.ones_like(idx.reshape(-1), dtype=torch.int32))
    if not c["grad"]:
        return {"idx": idx, "weights": w, "counts": counts}
    grad = torch.autograd.grad(w, z, c["gw"])[0].to(c["logits"].dtype)
    return {"idx": idx, "weights": w.detach(), "counts": counts, "grad": grad}


def _losses(c):
    if own:
        balance, z2 = _pkg().router_losses(c["logits"], c["idx"], scoring=c["scoring"], mask=c["m"], per_sequence=c["per_sequence"])
        grad = torch.autograd.grad([balance, z2], [c["logits"]], c["grads"])[0]
        return {"balance": balance.detach(), "z": z2.detach(), "grad": grad}
    z = c["logits"].detach().float().requires_grad_(True)
    B, S, E = z.shape
    m = torch.ones(B, S, device=z.device) if c["m"] is None else c["m"].float()
    top = z.amax(dim=2, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=2, keepdim=True)
    p = e / total
    if c["scoring"] == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        p = s / s.sum(dim=2, keepdim=True)
    z2 = ((torch.log(total) + top)[:, :, 0].square() * m).sum() / m.sum()
    hits = torch.zeros_like(z.detach()).scatter_(2, c["idx"], 1.0) * m[:, :, None]
    dims = 1 if c["per_sequence"] else (0, 1)
    n = m.sum(dim=dims)
    n1 = n.clamp(min=1)[..., None]
    each = ((hits.sum(dim=dims) * (E / c["k"]) / n1) * ((p * m[:, :, None]).sum(dim=dims) / n1)).sum(-1)
    balance = each.sum() / (n > 0).sum().clamp(min=1)
    grad = torch.autograd.grad([balance, z2], [z], c["grads"])[0].to(c["logits"].dtype)
    return {"balance": balance.detach(), "z": z2.detach(), "grad": grad}


def _rows(x):
    """x as the product reads it: codes of e4m3 with a scale per row and block of 128, as the values they stand for, in fp32."""
    K = x.shape[-1]
    p = torch.nn.functional.pad(x.float(), (0, -K % 128)).unflatten(-1, (-1, 128))
    amax = p.abs().amax(dim=-1, keepdim=True).clamp(min=2.0 ** -100)
    codes = torch.div(p * 448.0, amax).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return (codes.float() * torch.div(amax, torch.full_like(amax, 448.0))).flatten(-2)[..., :K]


def _values(codes, scale):
    """The values that the weights' codes stand for, in fp32."""
    N, K = codes.shape[-2:]
    return codes.float() * scale.repeat_interleave(128, dim=-2)[..., :N, :].repeat_interleave(128, dim=-1)[..., :K]


def _linear(c):
    if own:
        y = _pkg().fp8_block_linear(c["x"], c["w"], c["ws"])
        return {"y": y.detach(), "grad": torch.autograd.grad(y, c["x"], c["gy"])[0]} if c["grad"] else {"y": y}
    w = _values(c["w"], c["ws"])
    y = (_rows(c["x"].detach()) @ w.t()).to(torch.bfloat16)
    return {"y": y, "grad": (_rows(c["gy"]) @ w).to(torch.bfloat16)} if c["grad"] else {"y": y}


def _experts(c):
    if own:
        return _pkg().moe_fp8_block(c["x"], c["idx"], c["weights"], c["gate_up"], c["gate_up_scale"], c["down"], c["down_scale"])
    T, E, k, I = c["T"], c["E"], c["k"], c["I"]
    flat = c["idx"].reshape(-1)
    order = flat.sort(stable=True).indices
    counts = torch.zeros(E, dtype=torch.int64, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    place = torch.empty_like(flat)
    place[order] = torch.arange(T * k, device=flat.device) - (counts.cumsum(0) - counts)[flat[order]]
    rows = torch.zeros(E, int(counts.max()), c["x"].shape[1], device=flat.device)
    rows[flat, place] = _rows(c["x"])[torch.arange(T * k, device=flat.device) // k]
    h = torch.bmm(rows, _values(c["gate_up"], c["gate_up_scale"]).transpose(1, 2))
    gate, up = h[..., :I], h[..., I:]
    h = _rows(gate / (1 + torch.exp(-gate)) * up)
    y = torch.bmm(h, _values(c["down"], c["down_scale"]).transpose(1, 2))[flat, place].view(T, k, -1)
    return (y * c["weights"][:, :, None]).sum(dim=1).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _quantised64(x):
    x = x.double()
    T, K = x.shape
    out = torch.empty_like(x)
    for k0 in range(0, K, 128):
        block = x[:, k0:k0 + 128]
        amax = torch.clamp(block.abs().max(dim=1, keepdim=True).values, min=2.0 ** -100)
        out[:, k0:k0 + 128] = torch.clamp(block * 448.0 / amax, -448, 448).to(torch.float8_e4m3fn).double() * (amax / 448.0)
    return out


def _weight64(codes, scale):
    w = codes.double()
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            w[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= scale[i, j].double()
    return w


def exact(case, seed):
    c = prepare(case, seed)
    if c["op"] == "route":
        z = c["logits"].detach().double()
        idx = _picks(z, c)
        s = torch.sigmoid(z) if c["scoring"] == "sigmoid" else torch.softmax(z, dim=1)
        raw = s.gather(1, idx)
        t = raw.sum(1, keepdim=True) + 1e-20
        norm = c["norm"] and c["k"] > 1
        counts = torch.bincount(idx.reshape(-1), minlength=c["E"]).int()
        out = {"idx": idx, "weights": 2.5 * raw / t if norm else 2.5 * raw, "counts": counts}
        if c["grad"]:
            gw = c["gw"].double() * 2.5
            up = gw / t - (gw * raw).sum(1, keepdim=True) / t ** 2 if norm else gw
            ds = torch.zeros_like(s).scatter_add_(1, idx, up)
            out["grad"] = ds * s * torch.sigmoid(-z) if c["scoring"] == "sigmoid" else s * (ds - (ds * s).sum(1, keepdim=True))
        return out
    if c["op"] == "losses":
        z = c["logits"].detach().double()
        B, S, E = z.shape
        m = torch.ones(B, S, dtype=torch.float64, device=z.device) if c["m"] is None else c["m"].double()
        lse = torch.logsumexp(z, dim=2)
        soft = torch.softmax(z, dim=2)
        p = soft if c["scoring"] == "softmax" else torch.softmax(torch.nn.functional.logsigmoid(z), dim=2)
        parts = [slice(b, b + 1) for b in range(B)] if c["per_sequence"] else [slice(0, B)]
        live = sum(1 for b in parts if float(m[b].sum()) > 0)
        grad, balance = 2e-3 * (lse * m / m.sum())[:, :, None] * soft, torch.zeros((), dtype=torch.float64, device=z.device)
        for b in parts:
            n = m[b].sum()
            if float(n) == 0:
                continue
            f = torch.bincount(c["idx"][b][m[b] > 0].reshape(-1), minlength=E).double() * E / (c["k"] * n)
            balance = balance + (f * (p[b] * m[b][:, :, None]).sum((0, 1)) / n).sum() / live
            d = 0.01 * p[b] * (f - (p[b] * f).sum(2, keepdim=True)) * (m[b] / n)[:, :, None] / live
            grad[b] += d if c["scoring"] == "softmax" else d * torch.sigmoid(-z[b])
        return {"balance": balance, "z": (lse ** 2 * m).sum() / m.sum(), "grad": grad}
    if c["op"] == "linear":
        w = _weight64(c["w"], c["ws"])
        out = {"y": _quantised64(c["x"].detach()) @ w.t()}
        if c["grad"]:
            out["grad"] = _quantised64(c["gy"]) @ w
        return out
    x, I = _quantised64(c["x"]), c["I"]
    out = torch.zeros_like(x)
    for e in range(c["E"]):
        t, j = (c["idx"] == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        h = x[t] @ _weight64(c["gate_up"][e], c["gate_up_scale"][e]).t()
        h = _quantised64(torch.nn.functional.silu(h[:, :I]) * h[:, I:])
        out.index_add_(0, t, c["weights"][t, j].double()[:, None] * (h @ _weight64(c["down"][e], c["down_scale"][e]).t()))
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4}.get(c.get("dtype"), 2)
    if c["op"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        b, f = T * E * size + T * k * 12 + E * 4, 10 * T * E
        return {"bytes": b + (T * k * 4 + T * E * size if c["grad"] else 0), "flops": f * (2 if c["grad"] else 1)}
    if c["op"] == "losses":
        n = c["B"] * c["S"]
        return {"bytes": 2 * n * c["E"] * size + n * c["k"] * 8, "flops": 20 * n * c["E"]}
    if c["op"] == "linear":
        T, N, K = c["T"], c["N"], c["K"]
        weights = N * K + 4 * (-(-N // 128)) * (-(-K // 128))
        return {"bytes": weights + 2 * T * (N + K) * (2 if c["grad"] else 1), "flops": 2 * T * N * K * (2 if c["grad"] else 1)}
    T, E, H, I, k = (c[n] for n in ("T", "E", "H", "I", "k"))
    hit = E * (1 - (1 - k / E) ** T)      # experts with a row, on average over even routing
    return {"bytes": hit * 3 * H * I * (1 + 4 / 128 ** 2) + 4 * T * H + 12 * T * k, "flops": 6 * T * k * H * I}
