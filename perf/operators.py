"""The layer norm and the orthogonalised update of gan_amd, case by case: what is timed and checked, and their plain forms.

    norm     y = (x - mean) / sqrt(var + eps) * w + b over the rows of (rows, width); "train" adds its gradients, "penalty"
             the gradients of the input gradient (what a gradient penalty differentiates)
    ortho    Newton-Schulz orthogonalisation: X = G / max(|G|, eps), then X <- a X + (b A + c A A) X with A = X X' five times
    muon     one step of the orthogonalising optimiser over a list of matrices: momentum, orthogonalisation, update
"""
import math
import random

import torch

own = False

EPS = 1e-5
COEFFS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NORM_EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01

# The matrices of the StyleGAN2 256x256 discriminator with base_dim 16: every convolution as (out, in * kh * kw).
DISC = (
    "16x3,16x144,32x144,32x16,32x288,64x288,64x32,64x576,128x576,128x64,128x1152,256x1152,256x128,256x2304,512x2304,512x256,"
    "512x4608,512x4608,512x4617,512x512"
)

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the latents in front of a mapping network at a per-GPU batch of 32: the smallest call, all latency
        {"name": "norm latents", "op": "norm", "pass": "forward", "rows": 32, "width": 128, "dtype": "f32"},
        # every pixel of a (64, 512, 32, 32) activation, sampling or evaluation
        {"name": "norm pixels", "op": "norm", "pass": "forward", "rows": 65536, "width": 512, "dtype": "bf16"},
        # an odd width in full precision, trained: output and all three gradients
        {"name": "norm train odd", "op": "norm", "pass": "train", "rows": 4099, "width": 1001, "dtype": "f32"},
        # a critic that normalises whole samples: (64, 128, 16, 16), trained in mixed precision
        {"name": "norm train samples", "op": "norm", "pass": "train", "rows": 64, "width": 32768, "dtype": "bf16"},
        # a gradient penalty through the same kind of layer, one stage deeper, full precision
        {"name": "norm penalty samples", "op": "norm", "pass": "penalty", "rows": 64, "width": 16384, "dtype": "f32"},
        # a gradient penalty through a layer that normalises pixels, mixed precision
        {"name": "norm penalty pixels", "op": "norm", "pass": "penalty", "rows": 16384, "width": 512, "dtype": "bf16"},
        # the first 3x3 convolution of a base_dim 16 network: launches are all it costs
        {"name": "ortho 16x144", "op": "ortho", "batch": 1, "m": 16, "n": 144, "dtype": "f32"},
        # the 512-channel 3x3 convolution
        {"name": "ortho 512x4608", "op": "ortho", "batch": 1, "m": 512, "n": 4608, "dtype": "f32"},
        # odd sizes, more rows than columns, a batch of them in bfloat16
        {"name": "ortho 3x1000x777 bf16", "op": "ortho", "batch": 3, "m": 1000, "n": 777, "dtype": "bf16"},
        # the wide end: a matrix four times as long as wide
        {"name": "ortho 2048x8192", "op": "ortho", "batch": 1, "m": 2048, "n": 8192, "dtype": "f32"},
        # the eight linear layers of a mapping network
        {"name": "muon mapping", "op": "muon", "shapes": ",".join(["128x128"] * 8), "nesterov": True},
        # a whole discriminator, one optimiser step
        {"name": "muon discriminator", "op": "muon", "shapes": DISC, "nesterov": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["norm", "norm", "ortho", "ortho", "muon"])
    if op == "norm":
        width = _log(rng, 16, 65536)
        rows = _log(rng, 1, max(1, min(131072, (1 << 24) // width)))
        return {"op": op, "pass": rng.choice(["forward", "train", "penalty"]), "rows": rows, "width": width, "dtype": rng.choice(["f32", "bf16"])}
    if op == "ortho":
        m, n = _log(rng, 16, 1500), _log(rng, 16, 6000)
        if rng.random() < 0.4:
            m, n = n, m
        batch = max(1, min(_log(rng, 1, 16), (1 << 23) // (m * n)))
        return {"op": op, "batch": batch, "m": m, "n": n, "dtype": rng.choice(["f32", "bf16"])}
    shapes = []
    for _ in range(rng.randint(2, 12)):
        shapes.append("%dx%d" % (_log(rng, 8, 512), _log(rng, 8, 512) * rng.choice([1, 9])))
    return {"op": op, "shapes": ",".join(shapes), "nesterov": rng.random() < 0.7}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _gradient(m, n, g, device):
    """What a weight's gradient looks like: a few strong directions over a broad rest."""
    k = min(16, m, n)
    strong = torch.randn(m, k, generator=g, device=device) @ torch.randn(k, n, generator=g, device=device)
    return (strong * 0.25 + torch.randn(m, n, generator=g, device=device) * 0.5) * 1e-3


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    if case["op"] == "norm":
        rows, width, dt = case["rows"], case["width"], _TYPES[case["dtype"]]
        x = torch.randn(rows, width, generator=g, device=device) * 1.5
        x += torch.randn(rows, 1, generator=g, device=device)  # rows have means of their own
        s = {
            "case": dict(case),
            "x": x.to(dt).requires_grad_(case["pass"] != "forward"),
            "w": (1 + 0.2 * torch.randn(width, generator=g, device=device)).requires_grad_(case["pass"] != "forward"),
            "b": (0.2 * torch.randn(width, generator=g, device=device)).requires_grad_(case["pass"] != "forward"),
        }
        if case["pass"] != "forward":
            s["g"] = torch.randn(rows, width, generator=g, device=device).to(dt).requires_grad_(case["pass"] == "penalty")
        if case["pass"] == "penalty":
            s["v"] = torch.randn(rows, width, generator=g, device=device).to(dt)
        return s
    if case["op"] == "ortho":
        m, n = case["m"], case["n"]
        return {"case": dict(case), "g": torch.stack([_gradient(m, n, g, device) for _ in range(case["batch"])]).to(_TYPES[case["dtype"]])}
    params, grads, bufs = [], [], []
    for m, n in _shapes(case):
        params.append(torch.randn(m, n, generator=g, device=device) * 0.02)
        grads.append(_gradient(m, n, g, device))
        bufs.append(_gradient(m, n, g, device) * 0.3)
    return {"case": dict(case), "params": params, "grads": grads, "bufs": bufs}


# ---- plain forms ------------------------------------------------------------------------------------------------
def _plain_stats(x):
    x = x.detach().float()
    d = x - x.mean(1, keepdim=True)
    r = (d.square().mean(1, keepdim=True) + EPS).rsqrt()
    return d * r, r


def _plain_project(u, xh):
    """u without its mean and its part along xh, row by row."""
    return u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True)


def _plain_norm(s):
    x, w, b, kind = s["x"], s["w"].detach(), s["b"].detach(), s["case"]["pass"]
    dt = x.dtype
    xh, r = _plain_stats(x)
    y = (xh * w + b).to(dt)
    if kind == "forward":
        return y
    g = s["g"].detach().float()
    h = g * w
    gx = r * _plain_project(h, xh)
    if kind == "train":
        return y, gx.to(dt), (g * xh).sum(0), g.sum(0)
    v = s["v"].float()
    pv = r * _plain_project(v, xh)  # the input gradient is linear and symmetric in h
    hx, vx = (h * xh).mean(1, keepdim=True), (v * xh).mean(1, keepdim=True)
    dot = (v * h).mean(1, keepdim=True) - v.mean(1, keepdim=True) * h.mean(1, keepdim=True) - vx * hx
    xg = r * _plain_project(-r * (v * hx + h * vx), xh) - r.square() * dot * xh
    return gx.to(dt), xg.to(dt), (w * pv).to(dt), (g * pv).sum(0)


def _plain_ortho(g):
    """(..., m, n) in 32 bits."""
    a, b, c = COEFFS
    wide = g.shape[-2] <= g.shape[-1]
    x = g if wide else g.transpose(-2, -1).contiguous()
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(NORM_EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x if wide else x.transpose(-2, -1).contiguous()


def _plain_muon(s):
    for p, g, buf in zip(s["params"], s["grads"], s["bufs"]):
        buf.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
        u = g * (1 - MOMENTUM) + buf * MOMENTUM if s["case"]["nesterov"] else buf
        p.mul_(1 - LR * DECAY).sub_(_plain_ortho(u), alpha=LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1])))
    return s["params"], s["bufs"]


# ---- the framework's calls --------------------------------------------------------------------------------------
def _own_norm(s):
    from gan_amd import functional as GF

    x, w, b, kind = s["x"], s["w"], s["b"], s["case"]["pass"]
    y = GF.layer_norm(x, (x.shape[1],), w, b, EPS)
    if kind == "forward":
        return y
    if kind == "train":
        return (y, *torch.autograd.grad(y, (x, w, b), s["g"]))
    (gx,) = torch.autograd.grad(y, x, s["g"], create_graph=True)
    return (gx, *torch.autograd.grad(gx, (x, s["g"], w), s["v"]))


def _own_ortho(s):
    from gan_amd import functional as GF

    return GF.orthogonalize(s["g"], steps=STEPS, coefficients=COEFFS, eps=NORM_EPS)


def _own_muon(s):
    from gan_amd.optim import muon_step

    muon_step(s["params"], s["grads"], s["bufs"], lr=LR, momentum=MOMENTUM, nesterov=s["case"]["nesterov"], weight_decay=DECAY,
              steps=STEPS, coefficients=COEFFS, eps=NORM_EPS)
    return s["params"], s["bufs"]


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_norm(state) if op == "norm" else _own_ortho(state) if op == "ortho" else _own_muon(state)
    if op == "norm":
        return _plain_norm(state)
    if op == "ortho":
        return _plain_ortho(state["g"].float()).to(state["g"].dtype)
    return _plain_muon(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def _ortho_flops(m, n):
    """Either every iteration on the matrix itself (its Gram matrix and that one's square are symmetric: half the products),
    or the polynomial built up on the Gram matrix and applied once."""
    m, n = min(m, n), max(m, n)
    return min(STEPS * (3 * m * m * n + m**3), 3 * m * m * n + (4 * STEPS - 3) * m**3)


def work(case):
    if case["op"] == "norm":
        size, e = case["rows"] * case["width"], 4 if case["dtype"] == "f32" else 2
        vec = 4 * case["width"]
        if case["pass"] == "forward":
            return {"bytes": 2 * size * e + 2 * vec, "flops": 8 * size}
        if case["pass"] == "train":  # x, g in; y, gx out
            return {"bytes": 4 * size * e + 4 * vec, "flops": 20 * size}
        return {"bytes": 6 * size * e + 2 * vec, "flops": 45 * size}  # x, g, v in; gx and the two gradients out
    if case["op"] == "ortho":
        m, n, e = case["m"], case["n"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * case["batch"] * m * n * e, "flops": case["batch"] * _ortho_flops(m, n)}
    size = sum(m * n for m, n in _shapes(case))
    return {"bytes": 5 * 4 * size, "flops": sum(_ortho_flops(m, n) for m, n in _shapes(case))}  # p, g, momentum in; p, momentum out


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------
def _exact_polar(g):
    """The iterates through the singular values' polynomial, Horner's way, on the smaller side's Gram matrix."""
    a, b, c = COEFFS
    g = g.double()
    x = g / torch.linalg.matrix_norm(g).clamp_min(NORM_EPS)[..., None, None]
    tall = x.shape[-2] > x.shape[-1]
    eye = torch.eye(min(x.shape[-2:]), dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        xt = x.mT.contiguous()
        gram = xt @ x if tall else x @ xt
        poly = a * eye + gram @ (b * eye + c * gram)
        x = x @ poly if tall else poly @ x
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ortho":
        return _exact_polar(s["g"])
    if case["op"] == "muon":
        params, bufs = [], []
        for p, g, buf in zip(s["params"], s["grads"], s["bufs"]):
            m = MOMENTUM * buf.double() + (1 - MOMENTUM) * g.double()
            u = MOMENTUM * m + (1 - MOMENTUM) * g.double() if case["nesterov"] else m
            step = LR * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            params.append((1 - LR * DECAY) * p.double() - step * _exact_polar(u))
            bufs.append(m)
        return params, bufs
    x, w, b = (s[k].detach().double().requires_grad_(True) for k in "xwb")
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * w + b
    if case["pass"] == "forward":
        return y.detach()
    g = s["g"].detach().double().requires_grad_(True)
    if case["pass"] == "train":
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), g))
    (gx,) = torch.autograd.grad(y, x, g, create_graph=True)
    return (gx.detach(), *torch.autograd.grad(gx, (x, g, w), s["v"].double()))
