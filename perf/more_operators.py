"""Measurable cases of two operators that stand around the products over 8-bit weights: the root-mean-square norm with the residual's
addition, whose rows leave in their own type, as codes of e4m3 with a scale per block of 128, or both; and the low-rank adapters of many
requests, added to a shared projection's result.

`listed()` names twelve cases, `draw(rng)` gives others of the same ranges, `prepare` makes what a program holds before the call,
`run` is one pass (the package's entry points where `own` is true, elementary torch operations otherwise), `exact` the same in 64
bits, `work` the bytes and operations a pass cannot do without."""
import importlib
import math

import torch

own = False


def listed():
    return [
        # serving, the next token of one sequence: the residual stream goes on, the norm leaves as the codes that the next product reads
        dict(name="norm_decode_1", op="norm", T=1, K=4096, dtype="bf16", wtype="bf16", residual=True, y=False, codes=True, grad=False),
        # serving, prompts of a whole batch: the same, bound by memory
        dict(name="norm_prefill_16384", op="norm", T=16384, K=4096, dtype="bf16", wtype="bf16", residual=True, y=False, codes=True, grad=False),
        # training in bf16, forward and backward, with the gradient that comes down the residual stream
        dict(name="norm_train_16384", op="norm", T=16384, K=2048, dtype="bf16", wtype="bf16", residual=True, y=True, codes=False, grad=True),
        # fine-tuning beside frozen 8-bit weights: the products read codes, the adapters and the router rows
        dict(name="norm_tune_8192", op="norm", T=8192, K=4096, dtype="bf16", wtype="f32", residual=True, y=True, codes=True, grad=True),
        # a model held in fp32, without a residual; a width that fills no block of 128
        dict(name="norm_f32_5003", op="norm", T=5003, K=1032, dtype="f32", wtype="f32", residual=False, y=True, codes=False, grad=True),
        # odd rows in fp16, which start at no boundary of 16 bytes
        dict(name="norm_odd_333", op="norm", T=333, K=1037, dtype="f16", wtype="f16", residual=True, y=True, codes=False, grad=True),
        # serving, the next token of one request that has an adapter, beside a square projection
        dict(name="lora_decode_1", op="lora", T=1, K=4096, N=4096, R=16, L=8, rows="mixed", base=True, grad=False),
        # serving, the next tokens of 64 requests, each with its own of 64 adapters, beside a wide projection
        dict(name="lora_decode_64", op="lora", T=64, K=4096, N=14336, R=16, L=64, rows="mixed", base=True, grad=False),
        # serving, a larger batch: some requests share an adapter, some have none
        dict(name="lora_decode_512", op="lora", T=512, K=2048, N=2816, R=16, L=32, rows="mixed", base=True, grad=False),
        # serving, prompts packed one after another, of different lengths, each with its adapter or none
        dict(name="lora_prompts_8192", op="lora", T=8192, K=4096, N=14336, R=32, L=8, rows="packed", base=True, grad=False),
        # fine-tuning three small adapters at once, widths that fill no tile: gradients of the input and of both factors
        dict(name="lora_tune_3001", op="lora", T=3001, K=1040, N=680, R=8, L=3, rows="packed", base=True, grad=True),
        # fine-tuning one adapter in a large step
        dict(name="lora_tune_16384", op="lora", T=16384, K=2048, N=2816, R=64, L=1, rows="one", base=True, grad=True),
    ]


def _log(rng, lo, hi, mult=1):
    """A multiple of `mult` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi // mult * mult, max(-(-lo // mult) * mult, round(v / mult) * mult)))


def draw(rng):
    if rng.random() < 0.5:
        codes = rng.random() < 0.5
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        T, K = _log(rng, 1, 8192), _log(rng, 64, 2048 if dtype == "f32" else 4096, 8 if codes or rng.random() < 0.5 else 1)
        y = not codes or rng.random() < 0.5
        return dict(op="norm", T=T, K=K, dtype=dtype, wtype=rng.choice([dtype, "f32"]), residual=rng.random() < 0.7, y=y, codes=codes,
                    grad=y and rng.random() < 0.4)
    L = rng.choice([1, 1, 2, 4, 8, 16, 32])
    R = rng.choice([r for r in (8, 16, 24, 32, 48, 64, 128) if L * r <= 512])
    return dict(op="lora", T=_log(rng, 1, 8192), K=_log(rng, 64, 4096, 8), N=_log(rng, 64, 4096, 8), R=R, L=L,
                rows="one" if L == 1 and rng.random() < 0.5 else rng.choice(["packed", "packed", "mixed"]), base=rng.random() < 0.7,
                grad=rng.random() < 0.4)


_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")     # noqa: E731
    c = dict(case)
    T, K = c["T"], c["K"]
    if c["op"] == "norm":
        t = _TYPES[c["dtype"]]
        # a residual stream: rows of different size, a few columns that stand out
        c["x"] = (rand(T, K) * (0.5 + rand(T, 1).abs())).to(t).requires_grad_(c["grad"])
        c["r"] = (rand(T, K) * (1 + 4 * (rand(K) > 2.5))).to(t).requires_grad_(c["grad"]) if c["residual"] else None
        c["w"] = (1 + 0.2 * rand(K)).to(_TYPES[c["wtype"]]).requires_grad_(c["grad"])
        c["gy"], c["gh"] = (rand(T, K).to(t), rand(T, K).to(t)) if c["grad"] else (None, None)
        return c
    N, R, L = c["N"], c["R"], c["L"]
    c["x"] = rand(T, K).to(torch.bfloat16).requires_grad_(c["grad"])
    c["a"] = (rand(L, R, K) / math.sqrt(K)).to(torch.bfloat16).requires_grad_(c["grad"])
    c["b"] = (rand(L, N, R) * 0.3).to(torch.bfloat16).requires_grad_(c["grad"])
    c["s"] = 0.5 + torch.rand(L, generator=g, device="cuda")
    c["bs"] = rand(T, N).to(torch.bfloat16) if c["base"] else None
    c["gy"] = rand(T, N).to(torch.bfloat16) if c["grad"] else None
    c["i"] = None
    if c["rows"] == "mixed":        # a row a request; those with -1 have no adapter
        c["i"] = torch.randint(-1 if L > 1 and T > 1 else 0, L, (T,), generator=g, device="cuda")
    elif c["rows"] == "packed":     # requests of different lengths, one after another; one of them has no adapter
        ends = (torch.rand(L, generator=g, device="cuda") * T).long().sort().values
        of = torch.randperm(L + 1, generator=g, device="cuda") - (1 if L > 1 else 0)
        c["i"] = of[torch.searchsorted(ends, torch.arange(T, device="cuda"), right=True)].clamp(max=L - 1)
    return c


# ------------------------------------------------------------------------------------------------ one pass
def run(c):
    return _norm(c) if c["op"] == "norm" else _lora(c)


def _pkg():
    return importlib.import_module("triton-kernel-fused_b200")


def _norm(c):
    out = {}
    if own:
        if c["codes"]:
            got = _pkg().rms_norm_fp8_block(c["x"], c["w"], residual=c["r"], eps=_EPS, return_norm=c["y"])
            out["codes"], out["scale"], got = got[0], got[1], list(got[2:])
        else:
            got = _pkg().rms_norm(c["x"], c["w"], residual=c["r"], eps=_EPS)
            got = [got] if c["r"] is None else list(got)
        y = got.pop(0) if c["y"] else None
        h = got.pop(0) if c["residual"] else None
        x, r, w = c["x"], c["r"], c["w"]
    else:
        x, w = c["x"].detach().float().requires_grad_(c["grad"]), c["w"].detach().float().requires_grad_(c["grad"])
        r, h, v = None, None, x
        if c["residual"]:
            r = c["r"].detach().float().requires_grad_(c["grad"])
            h = x + r
            # the norm is of the stream as it goes on, in its own type
            v = h + (h.detach().to(c["x"].dtype).float() - h.detach())
        y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + _EPS) * w
        if c["codes"]:
            p = torch.nn.functional.pad(y.detach(), (0, -c["K"] % 128)).unflatten(-1, (-1, 128))
            amax = p.abs().amax(dim=-1, keepdim=True).clamp(min=2.0 ** -100)
            out["codes"] = torch.div(p * 448.0, amax).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).flatten(-2)[:, :c["K"]].contiguous()
            out["scale"] = torch.div(amax, torch.full_like(amax, 448.0))[..., 0]
    t = c["x"].dtype
    if c["grad"]:
        outs, gs = ([y], [c["gy"].to(y.dtype)]) if h is None else ([y, h], [c["gy"].to(y.dtype), c["gh"].to(h.dtype)])
        into = [x, w] if r is None else [x, r, w]
        grads = torch.autograd.grad(outs, into, gs)
        out["gx"], out["gw"] = grads[0].to(t), grads[-1].to(c["w"].dtype)
        if r is not None:
            out["gr"] = grads[1].to(t)
    if y is not None and c["y"]:
        out["y"] = y.detach().to(t)
    if h is not None:
        out["h"] = h.detach().to(t)
    return out


def _lora(c):
    if own:
        y = _pkg().lora_linear(c["x"], c["a"], c["b"], index=c["i"], scaling=c["s"], base=c["bs"])
        if not c["grad"]:
            return {"y": y}
        gx, ga, gb = torch.autograd.grad(y, [c["x"], c["a"], c["b"]], c["gy"])
        return {"y": y.detach(), "gx": gx, "ga": ga, "gb": gb}
    T, L, R, N = c["T"], c["L"], c["R"], c["N"]
    x, a, b = (c[n].detach().float().requires_grad_(c["grad"]) for n in ("x", "a", "b"))
    # all adapters side by side, a row's own scaled and the others times zero
    index = torch.zeros(T, dtype=torch.int64, device=x.device) if c["i"] is None else c["i"]
    of = (index[:, None] == torch.arange(L, device=x.device)).float() * c["s"]
    v = (x @ a.reshape(L * R, -1).t()) * of.repeat_interleave(R, dim=1)
    y = v @ b.transpose(1, 2).reshape(L * R, N)
    if c["bs"] is not None:
        y = y + c["bs"].float()
    out = {"y": y.detach().to(torch.bfloat16)}
    if c["grad"]:
        out["gx"], out["ga"], out["gb"] = (t.to(torch.bfloat16) for t in torch.autograd.grad(y, [x, a, b], c["gy"].float()))
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    c = prepare(case, seed)
    if c["op"] == "norm":
        x, w, K, t = c["x"].detach().double(), c["w"].detach().double(), c["K"], c["x"].dtype
        h = x if c["r"] is None else x + c["r"].detach().double()
        v = h if c["r"] is None else h.to(t).double()
        rstd = (v.square().sum(1, keepdim=True) / K + _EPS).rsqrt()
        n = v * rstd
        y, out = n * w, {}
        if c["codes"]:       # what the codes are the nearest to
            blocks = torch.nn.functional.pad(y, (0, -K % 128)).view(c["T"], -1, 128)
            amax = torch.clamp(blocks.abs().max(dim=2).values, min=2.0 ** -100)
            out["codes"] = (blocks * (448.0 / amax)[:, :, None]).view(c["T"], -1)[:, :K].contiguous()
            out["scale"] = amax / 448.0
        if c["grad"]:
            gy = c["gy"].double()
            d = gy * w
            gx = rstd * (d - n * (d * n).sum(1, keepdim=True) / K)
            if c["r"] is not None:
                gx = gx + c["gh"].double()
                out["gr"] = gx
            out["gx"], out["gw"] = gx, (gy * n).sum(0)
        if c["y"]:
            out["y"] = y
        if c["r"] is not None:
            out["h"] = h
        return out
    x, a, b = (c[n].detach().double() for n in ("x", "a", "b"))
    y = torch.zeros(c["T"], c["N"], dtype=torch.float64, device=x.device) if c["bs"] is None else c["bs"].double()
    gx, ga, gb = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    index = torch.zeros(c["T"], dtype=torch.int64, device=x.device) if c["i"] is None else c["i"]
    for j in range(c["L"]):
        rows = (index == j).nonzero().flatten()
        s, v = float(c["s"][j].double()), x[rows] @ a[j].t()
        y[rows] += s * (v @ b[j].t())
        if c["grad"]:
            g = c["gy"].double()[rows]
            u = s * (g @ b[j])
            gx[rows], ga[j], gb[j] = u @ a[j], u.t() @ x[rows], s * (g.t() @ v)
    return {"y": y, "gx": gx, "ga": ga, "gb": gb} if c["grad"] else {"y": y}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    T, K = c["T"], c["K"]
    if c["op"] == "norm":
        size, n = {"bf16": 2, "f16": 2, "f32": 4}[c["dtype"]], T * K
        b = n * size * (1 + 2 * c["residual"] + c["y"]) + (n + 4 * T * -(-K // 128) if c["codes"] else 0)
        if c["grad"]:        # the gradients of the norm and of the stream and the stream itself in, the gradient of both inputs out
            b += n * size * (3 + c["residual"])
        return {"bytes": b, "flops": n * (20 if c["grad"] else 6)}
    N, R, L = c["N"], c["R"], c["L"]
    hit = 1 if c["rows"] == "one" else L * (1 - (1 - 1 / L) ** T) if c["rows"] == "mixed" else L
    b, f = 2 * T * (K + N * (2 if c["base"] else 1)) + 2 * hit * R * (K + N), 2 * T * R * (K + N)
    if c["grad"]:       # the gradient of the result in, that of the input out, the input once more; those of the factors out
        b, f = b + 2 * T * (N + 2 * K) + 2 * L * R * (K + N), 3 * f
    return {"bytes": b, "flops": f}
