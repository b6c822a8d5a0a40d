"""Cases of the train step's layer norm and of its orthogonalised matrix updates.

Two families of operators, each in a plain form (elementary torch operations in 32 bits) and as the
package's kernels:

  norm   y = (x - mean(x)) / sqrt(var(x) + eps) * w + b over the last axis, and its backward pass
         (dx, and dw / db summed over the rows) -- phoneme_contrast_amd.layers.layer_norm
  orth   Newton-Schulz orthogonalisation of matrices: X = x / (|x|_F + eps), then `STEPS` times
         X <- a X + (b A + c A A) X with A = X X^T (the shorter side) --
         phoneme_contrast_amd.optim.orthogonalize
  muon   the update of a list of weight matrices by their orthogonalised momentum --
         phoneme_contrast_amd.optim.muon_step
"""
import math

import torch

own = False

EPS_NORM, EPS_ORTH = 1e-5, 1e-7
STEPS, COEF = 5, (3.4445, -4.7750, 2.0315)
LR, MOMENTUM, DECAY = 0.02, 0.95, 1e-2
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# weight matrices of the two networks (convolutions as [out, in, kh, kw], the projection last)
CNN_SMALL = "32x1x3x3,32x32x3x3,64x32x3x3,64x64x3x3,128x64x3x3,128x128x3x3,128x128"
CNN_DEEP = ("64x1x7x7,64x64x3x3,64x64x3x3,128x64x3x3,128x128x3x3,128x64x1x1,256x128x3x3,256x256x3x3,256x128x1x1,"
            "512x256x3x3,512x512x3x3,512x256x1x1,128x512")


def listed():
    return [
        # one clip's embedding at inference: latency alone
        {"name": "norm_infer_1x128_f32", "op": "norm", "rows": 1, "dim": 128, "type": "f32", "pad": 0, "train": False},
        # the projection head in training: the default batch (6 classes x 2 samples x 2 views), and the benchmark's
        {"name": "norm_train_24x128_f32", "op": "norm", "rows": 24, "dim": 128, "type": "f32", "pad": 0, "train": True},
        {"name": "norm_train_4096x128_f32", "op": "norm", "rows": 4096, "dim": 128, "type": "f32", "pad": 0, "train": True},
        # odd sizes, rows that are slices of a wider buffer
        {"name": "norm_train_1003x1537_bf16", "op": "norm", "rows": 1003, "dim": 1537, "type": "bf16", "pad": 7, "train": True},
        # token activations: a forward pass, and the largest training call
        {"name": "norm_infer_8192x5120_f16", "op": "norm", "rows": 8192, "dim": 5120, "type": "f16", "pad": 0, "train": False},
        {"name": "norm_train_16384x4096_bf16", "op": "norm", "rows": 16384, "dim": 4096, "type": "bf16", "pad": 0, "train": True},
        # the projection's gradient; the deepest convolution's; a batch of tall matrices of odd sizes; a square one
        {"name": "orth_128x128_f32", "op": "orth", "batch": 1, "rows": 128, "cols": 128, "type": "f32"},
        {"name": "orth_512x4608_f32", "op": "orth", "batch": 1, "rows": 512, "cols": 4608, "type": "f32"},
        {"name": "orth_6x1000x333_bf16", "op": "orth", "batch": 6, "rows": 1000, "cols": 333, "type": "bf16"},
        {"name": "orth_4096x4096_bf16", "op": "orth", "batch": 1, "rows": 4096, "cols": 4096, "type": "bf16"},
        # one optimiser step of every matrix of cnn_small and of cnn_deep
        {"name": "muon_cnn_small", "op": "muon", "shapes": CNN_SMALL, "nesterov": True},
        {"name": "muon_cnn_deep", "op": "muon", "shapes": CNN_DEEP, "nesterov": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "orth", "muon"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        dim = _log(rng, 1, 16384)
        return {"op": "norm", "rows": _log(rng, 1, min(65536, (1 << 26) // dim)), "dim": dim, "type": kind,
                "pad": rng.choice([0, 0, 0, 1, 8, 64]), "train": rng.random() < 0.6}
    if op == "orth":
        short = _log(rng, 1, 2048)
        long = _log(rng, short, 8192)
        batch = _log(rng, 1, max(1, min(16, (1 << 23) // (short * long))))
        rows, cols = (short, long) if rng.random() < 0.5 else (long, short)
        return {"op": "orth", "batch": batch, "rows": rows, "cols": cols, "type": kind}
    shapes, flops = [], 0
    for _ in range(rng.randint(1, 24)):
        out, cin, k = _log(rng, 2, 768), _log(rng, 1, 512), rng.choice([1, 3, 3, 5])
        flops += _orth_work(out, cin * k * k)
        if shapes and flops > 4e11:
            break
        shapes.append("%dx%d" % (out, max(2, cin)) if k == 1 else "%dx%dx%dx%d" % (out, cin, k, k))
    return {"op": "muon", "shapes": ",".join(shapes), "nesterov": rng.random() < 0.7}


def _gradients(shape, gen):
    """A matrix (or a batch) with the spectrum of a minibatch gradient: errors times inputs, summed over a few hundred
    samples whose directions are far from evenly spread, and some noise of the summation."""
    *batch, rows, cols = shape
    n = 256
    err = torch.randn(*batch, n, rows, device="cuda", generator=gen)
    act = torch.randn(*batch, n, cols, device="cuda", generator=gen)
    weight = torch.arange(1, n + 1, device="cuda").float().pow(-0.5)
    g = (err * weight[:, None]).transpose(-1, -2).contiguous() @ act
    return 1e-3 / n * (g + 0.1 * torch.randn(*batch, rows, cols, device="cuda", generator=gen))


def _shapes(case):
    return [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split(",")]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "norm":
        rows, dim, dt = case["rows"], case["dim"], TYPES[case["type"]]
        scale = torch.exp(0.5 * torch.randn(dim, device="cuda", generator=gen))
        shift = torch.randn(dim, device="cuda", generator=gen)
        x = torch.randn(rows, dim + case["pad"], device="cuda", generator=gen)
        x[:, :dim] = x[:, :dim] * scale + shift
        s = {"case": case, "x": x.to(dt)[:, :dim],
             "w": (1 + 0.1 * torch.randn(dim, device="cuda", generator=gen)).to(dt),
             "b": (0.1 * torch.randn(dim, device="cuda", generator=gen)).to(dt)}
        if case["train"]:
            s["dy"] = (0.01 * torch.randn(rows, dim, device="cuda", generator=gen)).to(dt)
            for k in ("x", "w", "b"):
                s[k].requires_grad_(True)
        return s
    if case["op"] == "orth":
        x = _gradients((case["batch"], case["rows"], case["cols"]), gen)
        return {"case": case, "x": (x * 100).to(TYPES[case["type"]])}
    s = {"case": case, "p": [], "g": [], "m": []}
    for shape in _shapes(case):
        flat = (shape[0], math.prod(shape[1:]))
        s["p"].append((torch.randn(flat, device="cuda", generator=gen) * (2.0 / flat[1]) ** 0.5).view(shape))
        s["g"].append(_gradients(flat, gen).view(shape))
        s["m"].append(_gradients(flat, gen).view(shape))
    return s


def _wide(x):
    """Rows of a few values in 64 bits (at two of them dx is what is left of a difference of 1e5 times its size)."""
    return x.double() if x.shape[-1] <= 32 else x.float()


def _plain_norm(x, w, b):
    d = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS_NORM)
    xhat = d * rstd
    return xhat * w + b, xhat, rstd


def _plain_orth(x):
    """[..., m, n] in 32 bits; works on the shorter side."""
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2).contiguous()
    norm = x.double().square().sum((-1, -2), keepdim=True).sqrt()
    x = (x.double() / (norm + EPS_ORTH)).float()
    a, b, c = COEF
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2).contiguous() if tall else x


def _adjusted(flat):
    return LR * 0.2 * math.sqrt(max(flat.shape))


@torch.no_grad()
def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        x, w = s["x"], s["w"]
        y, xhat, rstd = _plain_norm(_wide(x), w.float(), s["b"].float())
        y = y.to(x.dtype)
        if not case["train"]:
            return y
        dy = _wide(s["dy"])
        g = dy * w.float()
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        return {"y": y, "dx": dx.to(x.dtype), "dw": (dy * xhat).sum(0).to(w.dtype), "db": dy.sum(0).to(w.dtype)}
    if case["op"] == "orth":
        return _plain_orth(s["x"].float()).to(s["x"].dtype)
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        m.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
        u = g * (1 - MOMENTUM) + m * MOMENTUM if case["nesterov"] else m
        o = _plain_orth(u.reshape(u.shape[0], -1))
        p.mul_(1 - LR * DECAY).sub_(o.view_as(p), alpha=_adjusted(o))
    return {"p": s["p"], "m": s["m"]}


def run(s):
    if not own:
        return _plain(s)
    case = s["case"]
    if case["op"] == "norm":
        from phoneme_contrast_amd.layers import layer_norm
        x, w, b = s["x"], s["w"], s["b"]
        y = layer_norm(x, (case["dim"],), w, b, EPS_NORM)
        if not case["train"]:
            return y
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if case["op"] == "orth":
        from phoneme_contrast_amd.optim import orthogonalize
        return orthogonalize(s["x"], ns_steps=STEPS, ns_coefficients=COEF, eps=EPS_ORTH)
    from phoneme_contrast_amd.optim import muon_step
    muon_step(s["p"], s["g"], s["m"], lr=LR, momentum=MOMENTUM, nesterov=case["nesterov"], weight_decay=DECAY,
              ns_steps=STEPS, ns_coefficients=COEF, eps=EPS_ORTH)
    return {"p": s["p"], "m": s["m"]}


def _orth_work(rows, cols):
    """The products of the definition, a symmetric one's half counted once."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)


def work(case):
    if case["op"] == "norm":
        size = 4 if case["type"] == "f32" else 2
        n = case["rows"] * case["dim"]
        if case["train"]:  # forward: x in, y out; backward: x and dy in, dx out; w and b in, dw and db out
            return {"bytes": size * (5 * n + 5 * case["dim"]), "flops": 20 * n}
        return {"bytes": size * (2 * n + 2 * case["dim"]), "flops": 8 * n}
    if case["op"] == "orth":
        size = 4 if case["type"] == "f32" else 2
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * size * n, "flops": case["batch"] * _orth_work(case["rows"], case["cols"])}
    flats = [(s[0], math.prod(s[1:])) for s in _shapes(case)]
    return {"bytes": sum(4 * 5 * r * c for r, c in flats), "flops": sum(_orth_work(r, c) + 8 * r * c for r, c in flats)}


def _exact_orth(x):
    """In 64 bits, by matrix-vector association: A is applied to X and to A X instead of being squared."""
    wide = x if x.shape[-2] <= x.shape[-1] else x.transpose(-1, -2).contiguous()
    wide = wide / (torch.linalg.vector_norm(wide, dim=(-2, -1), keepdim=True) + EPS_ORTH)
    for _ in range(STEPS):
        gram = torch.matmul(wide, wide.transpose(-1, -2).contiguous())
        once = torch.matmul(gram, wide)
        wide = COEF[0] * wide + COEF[1] * once + COEF[2] * torch.matmul(gram, once)
    return wide if x.shape[-2] <= x.shape[-1] else wide.transpose(-1, -2).contiguous()


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w, b = (s[k].detach().double() for k in ("x", "w", "b"))
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS_NORM)
        unit = (x - mean) / sd
        y = torch.addcmul(b, unit, w)
        if not case["train"]:
            return y
        dy = s["dy"].double()
        up = dy * w
        dx = (up - up.mean(-1, keepdim=True) - unit * (up * unit).mean(-1, keepdim=True)) / sd
        return {"y": y, "dx": dx, "dw": torch.sum(dy * unit, 0), "db": torch.sum(dy, 0)}
    if case["op"] == "orth":
        return _exact_orth(s["x"].double())
    new_p, new_m = [], []
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        m2 = MOMENTUM * m.double() + (1 - MOMENTUM) * g.double()
        u = (1 - MOMENTUM) * g.double() + MOMENTUM * m2 if case["nesterov"] else m2
        o = _exact_orth(u.reshape(u.shape[0], -1)).reshape(u.shape)
        step = LR * 0.2 * max(u.shape[0], u.numel() // u.shape[0]) ** 0.5
        new_p.append((1 - LR * DECAY) * p.double() - step * o)
        new_m.append(m2)
    return {"p": new_p, "m": new_m}
