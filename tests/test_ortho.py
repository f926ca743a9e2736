"""functional.orthogonalize, optim.muon_step and optim.FlatMuon against the definition in 64 bits.

Bounds.  Products carry 22 bits of every factor (2^-22 relative to its largest entries) and fp32 sums, so a step adds an error of
a few 2^-22 of the iterate's norm; what the first steps add is amplified with the smallest singular values, by up to a = 3.4445
a step (485 in five).  For inputs whose singular values lie within a factor of 30 (Gaussian matrices a little off square, a few
strong directions over a broad rest) all of them are in the flat part after five steps, and the amplification of the error
relative to the value stays within that factor: 30 * 5 * 2^-22 = 3.6e-5 in the 2-norm, 1e-4 is asked.  A matrix of another kind
is held to 485 * 5 * 2^-22 = 6e-4.  bfloat16 results are rounded once, 2^-8 of the value each (2^-9 and less on average)."""
import math

import pytest
import torch

from conftest import rel_err

COEFFS = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def definition(g, steps=5, coefficients=COEFFS, eps=1e-7, on="cpu"):
    a, b, c = coefficients
    x = g.detach().double().to(on)
    x = x / torch.linalg.matrix_norm(x).clamp_min(eps)[..., None, None]
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    for _ in range(steps):
        gram = x @ x.mT.contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def make(m, n, dev, seed=0, dt=torch.float32, kind="gauss"):
    gen = torch.Generator(device="cpu").manual_seed(seed + 31 * m + n)
    x = torch.randn(m, n, generator=gen)
    if kind == "strong":
        x = x + 4 * torch.randn(m, 2, generator=gen) @ torch.randn(2, n, generator=gen)
    elif kind == "scaled":
        x = x * torch.logspace(0, -3, m)[:, None]
    elif kind == "lowrank":
        k = max(1, min(m, n) // 3)
        x = torch.randn(m, k, generator=gen) @ torch.randn(k, n, generator=gen)
    return x.to(dt).to(dev)


SIZES = [(1, 1), (1, 7), (9, 1), (2, 3), (16, 144), (144, 16), (63, 65), (64, 64), (65, 200), (200, 129), (128, 128), (130, 1000), (777, 300), (512, 1300), (257, 2304), (64, 512), (1024, 20), (97, 128), (128, 160), (33, 500), (96, 310)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", SIZES)
def test_against_the_definition(dev, m, n):
    from gan_amd import functional as GF

    for kind, lim in (("gauss", 1e-4), ("strong", 1e-4), ("scaled", 6e-4), ("lowrank", 6e-4)):
        if kind == "gauss" and m == n and m > 2:
            lim = 6e-4  # the smallest singular values of a square Gaussian matrix lie far below the others
        g = make(m, n, dev, kind=kind)
        got = GF.orthogonalize(g)
        assert got.shape == g.shape and got.dtype == torch.float32
        assert rel_err(got, definition(g)) < lim, kind
        bf = g.bfloat16()
        got = GF.orthogonalize(bf)
        assert got.dtype == torch.bfloat16
        assert rel_err(got, definition(bf)) < lim + 2.0**-8, kind


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1990, 33000), (2048, 8192), (1030, 4100), (500, 4610), (3, 1000, 1777), (9, 260, 2000), (20000, 3, 5), (100000, 40)])
def test_large_ones(dev, shape):
    """Sizes at which the larger tiles run, whole and with a part of one at the end, with their sums cut in slices and not; many
    matrices at once, and very long ones.  (The reference runs on the device, in 64 bits.)"""
    from gan_amd import functional as GF

    torch.manual_seed(5)
    g = torch.randn(shape, device=dev)
    if shape[-1] > 5:
        g += 4 * torch.randn(*shape[:-1], 2, device=dev) @ torch.randn(*shape[:-2], 2, shape[-1], device=dev)
    want = definition(g, on=dev)
    lim = 1e-4 if shape[-1] > 5 else 6e-4
    assert rel_err(GF.orthogonalize(g), want) < lim
    del want
    g = g.bfloat16()
    assert rel_err(GF.orthogonalize(g), definition(g, on=dev)) < lim + 2.0**-8


@pytest.mark.gpu
def test_two_calls_at_once(dev):
    """Calls on two streams, neither waiting for the other, leave the bits of calls one after another."""
    from gan_amd import functional as GF

    xs = [make(300, 2300, dev, seed=1), make(512, 900, dev, seed=2)]
    want = [GF.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, (x, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[k].append(GF.orthogonalize(x))
    torch.cuda.synchronize()
    for w, all_of in zip(want, got):
        assert all(torch.equal(w, y) for y in all_of)


@pytest.mark.gpu
def test_batches_scales_layouts(dev):
    from gan_amd import functional as GF

    g = torch.stack([make(48, 100, dev, seed=k) * 10.0 ** (6 * k - 12) for k in range(5)])  # 1e-12 ... 1e12
    got = GF.orthogonalize(g)
    want = definition(g)
    for k in range(5):
        assert rel_err(got[k], want[k]) < 1e-4, k
    assert torch.equal(GF.orthogonalize(g[3]), got[3])  # the same bits alone and in a batch
    assert torch.equal(GF.orthogonalize(g.view(5, 1, 48, 100)), got.view(5, 1, 48, 100))
    t = make(90, 70, dev)
    assert torch.equal(GF.orthogonalize(t.t()), GF.orthogonalize(t.t().contiguous()))  # strided
    off = torch.cat([torch.zeros(1, device=dev), t.flatten()])[1:].view(90, 70)  # not on a 16-byte boundary
    assert torch.equal(GF.orthogonalize(off), GF.orthogonalize(t))
    huge = make(20, 30, dev) * 1e25  # squares leave fp32
    assert rel_err(GF.orthogonalize(huge), definition(huge)) < 1e-4
    tiny = make(20, 30, dev) * 1e-9  # below eps: divided by eps
    assert rel_err(GF.orthogonalize(tiny), definition(tiny)) < 1e-4
    for shape in ((0, 4, 4), (3, 0, 5), (3, 5, 0)):
        assert GF.orthogonalize(torch.empty(shape, device=dev)).shape == shape


@pytest.mark.gpu
def test_zeros_and_values_that_are_not_finite(dev):
    from gan_amd import functional as GF

    g = torch.stack([make(70, 90, dev, seed=k) for k in range(6)])
    want = GF.orthogonalize(g)
    bad = g.clone()
    bad[1] = 0
    bad[2, 5, 7] = float("nan")
    bad[4, 69, 0] = float("inf")
    got = GF.orthogonalize(bad)
    for k in (0, 3, 5):
        assert torch.equal(got[k], want[k])
    assert torch.equal(got[1], torch.zeros_like(got[1]))
    assert torch.isnan(got[2]).all() and torch.isnan(got[4]).all()
    half = make(40, 60, dev)
    half[10:20] = 0  # rows of zeros stay zeros
    assert torch.equal(GF.orthogonalize(half)[10:20], torch.zeros(10, 60, device=dev))


@pytest.mark.gpu
@pytest.mark.parametrize("steps,coefficients", [(1, COEFFS), (2, COEFFS), (3, COEFFS), (8, COEFFS), (6, (2.0, -1.5, 0.5)), (12, (1.5, -0.5, 0.0)), (1, (1.0, 0.0, 0.0))])
def test_steps_and_coefficients(dev, steps, coefficients):
    """(the cubic and quintic iterations that converge to the polar factor too; (1, 0, 0) is the normalisation alone)"""
    from gan_amd import functional as GF

    for m, n in ((40, 150), (100, 60), (128, 700)):
        g = make(m, n, dev, kind="strong")
        want = definition(g, steps, coefficients)
        lim = 30 * (steps + 1) * 2.0**-22
        assert rel_err(GF.orthogonalize(g, steps=steps, coefficients=coefficients), want) < lim
        assert rel_err(GF.orthogonalize(g.bfloat16(), steps=steps, coefficients=coefficients), definition(g.bfloat16(), steps, coefficients)) < lim + 2.0**-8
    if steps == 12:
        x = GF.orthogonalize(make(40, 4000, dev), steps=12, coefficients=coefficients)
        assert rel_err(x @ x.t(), torch.eye(40)) < 1e-4  # converged


def step_ref(p, g, buf, lr, momentum, nesterov, wd, scaling, steps=5):
    p, g, buf = (t.detach().double().cpu() for t in (p, g, buf))
    m, n = p.shape[0], p[0].numel()
    buf = momentum * buf + (1 - momentum) * g
    u = momentum * buf + (1 - momentum) * g if nesterov else buf
    s = {None: max(1, m / n) ** 0.5, "original": max(1, m / n) ** 0.5, "match_rms_adamw": 0.2 * max(m, n) ** 0.5, "none": 1.0}[scaling]
    return (1 - lr * wd) * p - lr * s * definition(u.reshape(m, n), steps).reshape(p.shape), buf


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,wd,scaling", [(True, 0.0, None), (False, 0.1, "original"), (True, 0.01, "match_rms_adamw"), (False, 0.0, "none")])
def test_muon_step(dev, nesterov, wd, scaling):
    from gan_amd.optim import muon_step

    shapes = [(16, 3, 1, 1), (64, 48), (48, 64), (1, 5), (200, 10, 3, 3), (8, 8), (0, 4), (300, 1)] + [(12, 5, 3, 3)] * 40  # more than one launch holds
    gen = torch.Generator(device="cpu").manual_seed(2)
    p, g, buf = ([torch.randn(s, generator=gen).to(dev) for s in shapes] for _ in range(3))
    want = [step_ref(*t, 0.02, 0.9, nesterov, wd, scaling) for t in zip(p, g, buf) if t[0].numel()]
    before = [t.clone() for t in p if t.numel()]
    muon_step(p, g, buf, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=wd, adjust_lr_fn=scaling)
    for a, b, m, (wp, wb) in zip([t for t in p if t.numel()], before, [t for t in buf if t.numel()], want):
        assert rel_err(m, wb) < 1e-6
        # the update alone: orthogonalize's bound, and the parameter's own rounding against it (p ~ 1, the update 0.02 and smaller)
        upd, upd_w = a.double().cpu() - b.double().cpu(), wp - b.double().cpu()
        assert float((upd - upd_w).norm()) <= 6e-4 * float(upd_w.norm()) + 2.0**-23 * float(b.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(64, 512), (1024, 20), (96, 288)], [(300, 520), (40, 64, 3, 3)] + [(12, 5, 3, 3)] * 40 + [(129, 128), (700, 90)]])
def test_muon_step_of_large_and_small(dev, shapes):
    """Lists that fit into LDS matrix by matrix, and that do not: a long one in several groups, small ones among the others."""
    from gan_amd.optim import muon_step

    gen = torch.Generator(device="cpu").manual_seed(3)
    p, g, buf = ([torch.randn(s, generator=gen).to(dev) for s in shapes] for _ in range(3))
    want = [step_ref(*t, 0.5, 0.9, True, 0.01, "original") for t in zip(p, g, buf)]
    before = [t.clone() for t in p]
    muon_step(p, g, buf, lr=0.5, momentum=0.9, weight_decay=0.01)
    for a, b, m, (wp, wb) in zip(p, before, buf, want):
        assert rel_err(m, wb) < 1e-6
        upd, upd_w = a.double().cpu() - b.double().cpu(), wp - b.double().cpu()  # (the bound of test_muon_step)
        assert float((upd - upd_w).norm()) <= 6e-4 * float(upd_w.norm()) + 2.0**-23 * float(b.norm())


@pytest.mark.gpu
def test_same_bits_other_stream_and_graph(dev):
    from gan_amd import functional as GF
    from gan_amd.optim import muon_step

    g = make(150, 700, dev)
    gb = torch.stack([make(33, 20, dev, seed=k, dt=torch.bfloat16) for k in range(3)])
    p0, b0 = make(150, 700, dev, seed=3), make(150, 700, dev, seed=4)

    def step():
        p, b = p0.clone(), b0.clone()
        muon_step([p], [g], [b], lr=0.1)
        return [GF.orthogonalize(g), GF.orthogonalize(gb), p, b]

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, held = [], []
    torch.cuda.synchronize()
    for _ in range(2):  # two graphs, each with its workspace
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step())
    for k in range(3):
        g.mul_(-1.5), gb.copy_(gb.flip(0))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for h in held:
            assert all(torch.equal(a, b) for a, b in zip(eager, h)), k


def adam_ref(p, g, m, v, t, lr, betas, eps):
    m.mul_(betas[0]).add_(g, alpha=1 - betas[0])
    v.mul_(betas[1]).addcmul_(g, g, value=1 - betas[1])
    p.addcdiv_(m / (1 - betas[0] ** t), (v / (1 - betas[1] ** t)).sqrt().add_(eps), value=-lr)


@pytest.mark.gpu
def test_flat_muon(dev):
    """make_optimizer("Muon"): matrices by muon_step's rule, the rest by Adam's, against both in 64 bits over four steps in which
    one matrix and one bias each skip a step; state_dict and back; frozen parameters."""
    from torch import nn

    from gan_amd.optim import FlatMuon, make_optimizer

    torch.manual_seed(0)

    def build():
        net = nn.Sequential(nn.Conv2d(3, 20, 3), nn.LayerNorm(20), nn.Linear(30, 11), nn.Conv2d(9, 1, 2), nn.Linear(6, 6, bias=False)).to(dev)
        net.register_parameter("scale", nn.Parameter(torch.ones(7, 1, 1, device=dev)))
        net[4].weight.requires_grad_(False)
        return net

    net = build()
    opt = make_optimizer("Muon", net, 0.05, {"weight_decay": 0.02, "momentum": 0.8, "adam_lr": 2e-3, "betas": [0.5, 0.9]})
    assert isinstance(opt, FlatMuon) and len(opt.param_groups) == 2
    params = list(net.parameters())
    ref = [p.detach().double().cpu().clone() for p in params]
    m, v = ([torch.zeros_like(r) for r in ref] for _ in range(2))
    is_matrix = [r.dim() >= 2 and min(r.shape[0], r[0].numel()) > 1 for r in ref]
    assert sum(is_matrix) == 3 and len(opt.param_groups[0]["params"]) == 3
    frozen = params[-2] if not params[-2].requires_grad else next(p for p in params if not p.requires_grad)
    held = frozen.detach().clone()
    for step in range(4):
        for i, (p, r) in enumerate(zip(params, ref)):
            if (step == 2 and i in (0, 1)) or not p.requires_grad:
                p.grad = None
                continue
            g = torch.randn(p.shape) * 10.0 ** (i - 3)
            p.grad = g.to(dev)
            if is_matrix[i]:
                r.copy_(step_ref(r, g, m[i], 0.05, 0.8, True, 0.02, None)[0])
                m[i].mul_(0.8).add_(g.double(), alpha=1 - 0.8)
            else:
                adam_ref(r, g.double(), m[i], v[i], step + 1, 2e-3, (0.5, 0.9), 1e-8)
        before = [p.detach().clone() for p in params]
        opt.step()
        for i, (p, r) in enumerate(zip(params, ref)):
            if step == 2 and i in (0, 1):
                assert torch.equal(p, before[i])
            elif p.requires_grad:
                # (p ~ 0.1 ... 1 with its own rounding; four updates of 0.05 x 1 / sqrt(n) an entry within 6e-4 of themselves)
                assert float((p.detach().double().cpu() - r).norm()) <= 1e-5 * float(r.norm()) + 4 * 6e-4 * 0.05 * math.sqrt(min(r.shape[0], r[0].numel()) if is_matrix[i] else 0), (step, i)
    assert torch.equal(frozen, held)
    # a second optimizer continues from the state
    saved = opt.state_dict()
    keys = [set(s) for s in saved["state"].values()]
    assert {"momentum_buffer"} in keys and {"step", "exp_avg", "exp_avg_sq"} in keys
    twin = build()
    twin.load_state_dict(net.state_dict())
    opt2 = make_optimizer("Muon", twin, 1.0, {})
    opt2.load_state_dict(saved)
    for p, q in zip(params, twin.parameters()):
        if p.requires_grad:
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
    opt.step(), opt2.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twin.parameters()))
    # a bad coefficient is refused at the step, other classes stay torch's
    assert isinstance(make_optimizer("Muon", nn.Linear(3, 3, bias=False), 0.1, {}), torch.optim.Muon)  # (not on the device)
    with pytest.raises(ValueError):
        make_optimizer("Muon", build(), 0.1, {"adjust_lr_fn": "x"})


@pytest.mark.gpu
def test_norm_penalty_and_step_together(dev):
    """What the operators are for: a critic that normalises whole samples, trained by WGAN-GP (its penalty differentiates the
    norm's backward) with the orthogonalised step.  Gradients against the same critic in 64 bits; the update against the
    rule; then the whole step replayed as a HIP graph against the eager one."""
    from torch import nn

    from gan_amd.losses import wgan_gp_regularizer
    from gan_amd.modelling.common import Conv2d, LayerNorm, LeakyReLU
    from gan_amd.optim import make_optimizer

    torch.manual_seed(5)

    class Critic(nn.Module):
        def __init__(self, conv, norm, act):
            super().__init__()
            self.conv, self.norm, self.act, self.head = conv(3, 24, 3, padding=1), norm((24, 8, 8)), act(0.2), nn.Linear(24 * 64, 1)

        def forward(self, x):
            return self.head(self.act(self.norm(self.conv(x))).flatten(1))[:, 0]

    net = Critic(Conv2d, LayerNorm, LeakyReLU).to(dev)
    with torch.no_grad():
        net.norm.weight.normal_(1, 0.3), net.norm.bias.normal_(0, 0.3)
    ref = Critic(nn.Conv2d, nn.LayerNorm, nn.LeakyReLU).double()
    ref.load_state_dict({k: t.double().cpu() for k, t in net.state_dict().items()})
    reals, fakes, alpha = torch.randn(6, 3, 8, 8), torch.randn(6, 3, 8, 8), torch.rand(6, 1, 1, 1)
    inter = (reals + alpha * (fakes - reals)).double().requires_grad_()
    (gx,) = torch.autograd.grad(ref(inter).sum(), inter, create_graph=True)
    penalty = (gx.flatten(1).norm(dim=1) - 1).square().mean() * 10
    (penalty + ref(fakes.double()).mean() - ref(reals.double()).mean()).backward()

    opt = make_optimizer("Muon", net, 0.02, {"weight_decay": 0.0})
    opt.zero_grad()
    real_rand = torch.rand
    try:
        torch.rand = lambda *a, **k: alpha.to(dev)
        loss = wgan_gp_regularizer(net, reals.to(dev), fakes.to(dev), None) + net(fakes.to(dev)).mean() - net(reals.to(dev)).mean()
    finally:
        torch.rand = real_rand
    loss.backward()
    for (name, p), q in zip(net.named_parameters(), ref.parameters()):
        assert rel_err(p.grad, q.grad) < 1e-4, name  # (fp32 convolutions of 27 and products of 1536 terms, twice differentiated)
    before = {n: p.detach().double().cpu().clone() for n, p in net.named_parameters()}
    opt.step()
    w = net.conv.weight
    want, _ = step_ref(before["conv.weight"], w.grad, torch.zeros_like(w), 0.02, 0.95, True, 0.0, None)
    upd = w.detach().double().cpu() - before["conv.weight"]
    assert float((upd - (want - before["conv.weight"])).norm()) <= 6e-4 * float((want - before["conv.weight"]).norm()) + 2.0**-23 * float(want.norm())
    del loss

    # ---- captured and replayed: a multilayer critic (library products: the same bits every time)
    def build():
        torch.manual_seed(9)
        return nn.Sequential(nn.Linear(40, 96), LayerNorm(96), nn.Tanh(), nn.Linear(96, 96), LayerNorm(96), nn.Tanh(), nn.Linear(96, 1)).to(dev)

    def trainer(net):
        opt = make_optimizer("Muon", net, 0.02, {"weight_decay": 0.01, "adam_lr": 1e-3})

        def step(x):
            opt.zero_grad()
            xi = x.detach().requires_grad_()
            (g,) = torch.autograd.grad(net(xi).sum(), xi, create_graph=True)
            ((g.norm(dim=1) - 1).square().mean() + net(x).mean()).backward()
            opt.step()

        return step

    nets = build(), build()
    eager, graphed = trainer(nets[0]), trainer(nets[1])
    batches = [torch.randn(32, 40, device=dev) for _ in range(7)]
    x = batches[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for b in batches[:3]:
            x.copy_(b)
            graphed(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed(x)
    for k, b in enumerate(batches):
        eager(b)
        if k >= 3:
            x.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            for p, q in zip(*(n.parameters() for n in nets)):
                assert rel_err(q, p) < 1e-4, k


@pytest.mark.gpu
@pytest.mark.parametrize("hip_graph", [False, True])
def test_trainer_with_muon(dev, hip_graph, tmp_path):
    """TrainConfig(optimizer="Muon"): the train step runs, eager and as HIP graphs, and a checkpoint continues with the same
    optimizer state."""
    from gan_amd.optim import FlatMuon
    from gan_amd.train_celeba import TrainConfig, Trainer

    torch.manual_seed(1)
    cfg = TrainConfig(model="dcgan", img_size=32, gen_kwargs={"base_dim": 16}, disc_kwargs={"base_dim": 16, "norm": "none"}, method="wgan",
                      regularizer="wgan-gp", batch_size=8, optimizer="Muon", optimizer_kwargs={"weight_decay": 0.0, "adam_lr": 1e-4}, lr=2e-3,
                      device="cuda", mixed_precision=True, hip_graph=hip_graph, graph_warmup=2)
    reals = torch.randn(8, 3, 32, 32, device=dev)
    a = Trainer(cfg, dev)
    assert isinstance(a.optim_d, FlatMuon) and isinstance(a.optim_g, FlatMuon)
    before = [p.detach().clone() for p in a.gen.parameters()]
    for _ in range(5):
        logs = a.train_step(lambda: reals)
        assert all(math.isfinite(float(v)) for v in logs.values())
    assert (a._graph is not None) == hip_graph and a.cfg.hip_graph == hip_graph  # (a capture that fails falls back)
    assert all(torch.isfinite(p).all() for p in a.disc.parameters())
    assert not any(torch.equal(p, q) for p, q in zip(a.gen.parameters(), before))
    path = str(tmp_path / "c.pt")
    a.save_checkpoint(path)
    b = Trainer(cfg, dev)
    b.load_checkpoint(path)
    for x, y in ((a.optim_g, b.optim_g), (a.optim_d, b.optim_d)):
        # (the arenas' padding between parameters belongs to no state)
        for p, q in zip(x.arena.params, y.arena.params):
            assert torch.equal(p, q)
            assert all(torch.equal(x.state[p][k], y.state[q][k]) for k in x.state[p])
    b.train_step(lambda: reals)


def test_refusals():
    from gan_amd import _lib
    from gan_amd import functional as GF
    from gan_amd.optim import muon_step

    x = torch.randn(4, 8)
    for call in (
        lambda: GF.orthogonalize(x),  # not on a ROCm device
        lambda: GF.orthogonalize(x[0]),
        lambda: GF.orthogonalize(x.half()),
        lambda: GF.orthogonalize(x.requires_grad_()),
    ):
        with pytest.raises(_lib.GanAmdError):
            call()
    x, flat = x.detach(), torch.randn(64)
    for args, kw in (
        (([x], [x.clone()], [x.clone()]), {}),  # not on a ROCm device
        (([x], [], [x]), {}),
        (([x[0]], [x[0]], [x[0]]), {}),
        (([x], [x.t()], [x]), {}),
        (([x.double()], [x], [x]), {}),
        (([x.t()], [x.t()], [x.t()]), {}),
        (([x, x], [x.clone(), x.clone()], [x.clone(), x.clone()]), {}),
        (([x], [x], [x.clone()]), {}),
        (([x], [x.clone()], [x]), {}),
        (([x], [x.clone()], [x.clone()]), dict(adjust_lr_fn="other")),
        (([flat[:32].view(4, 8), flat[31:63].view(4, 8)], [x.clone(), x.clone()], [x.clone(), x.clone()]), {}),
        (([flat[:32].view(4, 8)], [flat[31:63].view(4, 8)], [x.clone()]), {}),
    ):
        with pytest.raises(_lib.GanAmdError):
            muon_step(*args, lr=0.1, **kw)
    # the C entries refuse before anything is launched
    import ctypes

    lib = _lib.load()
    p = 4096  # never read

    def mats(*rows):
        return (_lib.Matrix * len(rows))(*rows)

    def run(m, steps=5, coeffs=COEFFS, eps=1e-7, dtype=0, ws=p, nbytes=1 << 40):
        return lib.gan_orthogonalize(ctypes.addressof(m), len(m), steps, *coeffs, eps, dtype, ws, nbytes, None)

    ok = mats((p, None, p, 300, 256, 1))
    tiny = mats((p, None, p, 4, 8, 1))  # fits into LDS: no workspace
    assert lib.gan_orthogonalize_workspace(ctypes.addressof(tiny), 1) == 0 and run(tiny, steps=0) != 0 and run(tiny, eps=0.0) != 0
    need = lib.gan_orthogonalize_workspace(ctypes.addressof(ok), 1)
    assert need > 0
    assert run(ok, steps=0) != 0 and run(ok, steps=101) != 0
    assert run(ok, eps=0.0) != 0 and run(ok, eps=float("nan")) != 0
    assert run(ok, eps=1e-31) != 0 and run(ok, eps=1e31) != 0
    assert run(ok, coeffs=(10.0, 0.0, 0.0)) != 0 and run(ok, coeffs=(float("nan"), 0.0, 0.0)) != 0
    assert run(ok, dtype=2) != 0
    assert run(ok, ws=None) != 0 and run(ok, nbytes=need - 1) != 0 and run(ok, ws=p + 16) != 0
    assert run(mats((None, None, p, 4, 8, 1))) != 0 and run(mats((p, None, None, 4, 8, 1))) != 0
    assert run(mats((p, p, p, 4, 8, 1))) != 0  # a momentum buffer without a step
    for rows, cols, batch in ((0, 8, 1), (4, -1, 1), (4, 8, -1), (1 << 21, 8, 1), (40000, 40000, 1), (1 << 20, 1024, 1), (4, 8, 1 << 31)):
        bad = mats((p, None, p, rows, cols, batch))
        assert lib.gan_orthogonalize_workspace(ctypes.addressof(bad), 1) < 0 and run(bad) != 0
    assert run(mats((p, None, p, 4, 8, 0))) == 0  # nothing to do
    assert lib.gan_orthogonalize(None, 1, 5, *COEFFS, 1e-7, 0, p, 1 << 40, None) != 0
    step = mats((p, p, p, 300, 256, 1))

    def muon(m, lr=0.1, mu=0.9, wd=0.0, scaling=1):
        return lib.gan_muon_step(ctypes.addressof(m), len(m), lr, mu, 1, wd, scaling, 5, *COEFFS, 1e-7, p, need - 1, None)

    assert muon(step, lr=-1.0) != 0 and muon(step, mu=1.0) != 0 and muon(step, wd=-1.0) != 0 and muon(step, scaling=3) != 0
    assert muon(ok) != 0  # no momentum buffer
    assert muon(step) != 0 and b"workspace" in lib.gan_amd_last_error()


@pytest.mark.gpu
def test_narrow_matrices_in_a_list(dev):
    """Up to 192 rows a matrix goes step by step in a list too: no less accurate than the same iteration in fp32 products, on the
    average of some that are wide enough for two iterations from one A (which leave 1.1 to 2.3 times that error, measured; step by
    step 0.6 to 0.8).  With no momentum, a step of 1 from zero is the orthogonalised gradient itself."""
    from gan_amd.optim import muon_step

    shapes = [(32, 288), (64, 288), (64, 576), (128, 576), (128, 1152), (340, 171), (150, 800), (300, 1000)]
    gen = torch.Generator(device="cpu").manual_seed(11)
    ratios, late = [], []
    for _ in range(3):
        g = [(0.25 * torch.randn(m, 16, generator=gen) @ torch.randn(16, n, generator=gen) + 0.5 * torch.randn(m, n, generator=gen)).to(dev) for m, n in shapes]
        p, buf = ([torch.zeros_like(t) for t in g] for _ in range(2))
        muon_step(p, g, buf, lr=1.0, momentum=0.0, nesterov=False, adjust_lr_fn="none")
        for got, t in list(zip(p, g))[:7]:
            want = definition(t)
            a, b, c = COEFFS
            x = t / t.norm() if t.shape[0] <= t.shape[1] else (t / t.norm()).t().contiguous()
            for _ in range(5):
                gram = x @ x.t().contiguous()
                x = a * x + (b * gram + c * (gram @ gram)) @ x
            x = x if t.shape[0] <= t.shape[1] else x.t()
            (ratios if t.shape[1] > 171 and t.shape[0] <= 128 else late).append(rel_err(-got, want) / rel_err(x, want))
    assert sum(ratios) / len(ratios) < 1.0 and sum(late) / len(late) < 1.0, (ratios, late)


def test_limits_of_a_batch():
    """What the calls refuse, the workspace query says by a negative number; what it gives a size for, they take."""
    import ctypes

    from gan_amd import _lib

    lib = _lib.load()

    def need(*sizes):
        m = (_lib.Matrix * len(sizes))(*((4096, None, 4096, *s) for s in sizes))
        return lib.gan_orthogonalize_workspace(ctypes.addressof(m), len(m)), lib.gan_orthogonalize(ctypes.addressof(m), len(m), 5, *COEFFS, 1e-7, 0, None, 0, None)

    assert need((8, 8, 1 << 22)) == (-1, need((8, 8, 1 << 22))[1]) and need((8, 8, 1 << 22))[1] != 0
    assert need((200, 200, 1 << 20))[0] < 0 and need((200, 200, 1 << 20))[1] != 0  # (16 blocks each)
    assert need((200, 200, 1), (8, 8, 1 << 22))[0] < 0
    for sizes in (((200, 200, (1 << 19) - 1),), ((64, 64, (1 << 22) - 1), (200, 200, 1)), ((1 << 20, 64, 511),), ((32768, 32704, 32),), ((64, 4096, 300),), ((640, 40960, 400),)):
        assert need(*sizes)[0] > 0 and need(*sizes)[1] != 0  # (no workspace given)
        assert b"workspace" in lib.gan_amd_last_error()
    m = (_lib.Matrix * 2)((4096, None, 4096, 8, 8, (1 << 22) - 1), (4096, None, 4096, 200, 100, 3))
    assert lib.gan_orthogonalize_workspace(ctypes.addressof(m), 1) == 0  # in LDS
    assert lib.gan_orthogonalize_workspace(ctypes.addressof(m), 2) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(200000, 8, 8), (20000, 70, 65)])
def test_large_batches(dev, shape):
    from gan_amd import functional as GF

    torch.manual_seed(3)
    g = torch.randn(shape, device=dev)
    got, want = GF.orthogonalize(g).double(), torch.cat([definition(t, on=dev) for t in g.split(50000)])
    # (the bound of a square Gaussian matrix; one in so many lies further off than a factor of 30, each is held to its own)
    assert float(((got - want).norm(dim=(1, 2)) / want.norm(dim=(1, 2))).max()) < 6e-4


@pytest.mark.gpu
def test_lists_beyond_one_launch(dev):
    """Two batches that a launch does not hold together."""
    import ctypes

    from gan_amd import _lib

    torch.manual_seed(4)
    g = [torch.randn(2200000, 2, 3, device=dev), torch.randn(2100000, 3, 1, device=dev)]
    out = [torch.empty_like(t) for t in g]
    m = (_lib.Matrix * 2)(*((t.data_ptr(), None, o.data_ptr(), t.shape[1], t.shape[2], t.shape[0]) for t, o in zip(g, out)))
    lib = _lib.load()
    assert lib.gan_orthogonalize_workspace(ctypes.addressof(m), 2) == 0
    assert lib.gan_orthogonalize(ctypes.addressof(m), 2, 5, *COEFFS, 1e-7, 0, None, 0, _lib.stream_of(g[0])) == 0
    for t, o in zip(g, out):
        want = torch.cat([definition(part, on=dev) for part in t.split(50000)])
        assert float(((o.double() - want).norm(dim=(1, 2)) / want.norm(dim=(1, 2))).max()) < 6e-4


@pytest.mark.gpu
def test_muon_step_is_seen_by_a_backward_that_waits(dev):
    """A parameter changed between a forward and its backward: autograd refuses, as for any other change in place."""
    from gan_amd.optim import muon_step

    p = torch.randn(12, 20, device=dev, requires_grad=True)
    buf = torch.zeros(12, 20, device=dev)
    g = torch.randn(12, 20, device=dev)
    x = torch.randn(5, 12, device=dev, requires_grad=True)
    y = (x @ p).sum()
    versions = p._version, buf._version, g._version
    muon_step([p], [g], [buf], lr=0.1)
    assert (p._version, buf._version, g._version) == (versions[0] + 1, versions[1] + 1, versions[2])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():  # (tensors without a version)
        q = torch.randn(12, 20, device=dev)
        muon_step([q], [g], [torch.zeros_like(q)], lr=0.1)
    assert torch.isfinite(q).all()


def test_dual_tensors_are_refused():
    """A tangent would be dropped without a word: both say that there is no derivative."""
    from torch.autograd import forward_ad

    from gan_amd import _lib
    from gan_amd import functional as GF
    from gan_amd.optim import muon_step

    with forward_ad.dual_level():
        x = torch.randn(4, 8)
        dual = forward_ad.make_dual(x.clone(), torch.ones_like(x))
        with pytest.raises(_lib.GanAmdError, match="no derivative"):
            GF.orthogonalize(dual)
        with torch.no_grad(), pytest.raises(_lib.GanAmdError, match="no derivative"):
            GF.orthogonalize(dual)
        for args in (([dual], [x], [x.clone()]), ([x], [dual], [x.clone()]), ([x], [x.clone()], [dual])):
            with pytest.raises(_lib.GanAmdError, match="no derivative"):
                muon_step(*args, lr=0.1)
        with pytest.raises(_lib.GanAmdError) as plain:
            GF.orthogonalize(x)
        assert "derivative" not in str(plain.value)  # (not on a ROCm device)


@pytest.mark.gpu
def test_modules_that_torch_muon_takes(dev):
    """Two-dimensional parameters only: every one of them goes by the rule of torch.optim.Muon, a head of one row too.  (torch's
    class runs on the CPU, its products in bfloat16: five steps of three roundings of 2^-8, a few times that after their
    amplification; a quarter of the update is asked.  Adam's update of a row of 30 would be 5 times the rule's.)"""
    from torch import nn

    from gan_amd.optim import make_optimizer

    torch.manual_seed(2)
    net = nn.Sequential(nn.Linear(20, 30, bias=False), nn.Linear(30, 1, bias=False), nn.Linear(1, 6, bias=False)).to(dev)
    twin = [nn.Parameter(p.detach().cpu().clone()) for p in net.parameters()]
    opt = make_optimizer("Muon", net, 0.05, {"weight_decay": 0.02, "momentum": 0.8})
    stock = torch.optim.Muon(twin, lr=0.05, weight_decay=0.02, momentum=0.8)
    assert len(opt.param_groups) == 1 and all(set(opt.state[p]) == {"momentum_buffer"} for p in net.parameters())
    ref = [p.detach().double().clone() for p in twin]
    m = [torch.zeros_like(r) for r in ref]
    for _ in range(3):
        for i, (p, q) in enumerate(zip(net.parameters(), twin)):
            q.grad = torch.randn(q.shape)
            p.grad = q.grad.to(dev)
        before = [p.detach().clone() for p in twin]
        opt.step(), stock.step()
        for i, (p, q) in enumerate(zip(net.parameters(), twin)):
            old = ref[i]
            ref[i], m[i] = step_ref(old, q.grad, m[i], 0.05, 0.8, True, 0.02, None)
            assert float((p.detach().double().cpu() - ref[i]).norm()) <= 1e-5 * float(ref[i].norm()) + 6e-4 * 0.05 * 3 * min(p.shape) ** 0.5
            step = q.detach().double() - before[i].double()
            assert float((step - (ref[i] - old)).norm()) <= 0.25 * float((ref[i] - old).norm())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(40, 150), (300, 1200), (200, 70), (1, 9), (512, 4608)])
def test_norms_far_below_eps(dev, m, n):
    """X = G / eps stays small through all steps, which then multiply by little more than a: three roundings of 2^-22 a step, 15 in
    all, 3.6e-6; 1e-5 is asked, whatever the norm.  In LDS and not, with sums in slices, as a batch beside matrices of other norms."""
    from gan_amd import functional as GF
    from gan_amd.optim import muon_step

    g = make(m, n, dev)
    g = g / g.norm()
    for norm, eps in ((1e-9, 1e-7), (1e-13, 1e-7), (1e-18, 1e-7), (1e-30, 1e-7), (1.0, 1e4), (1e-3, 1e30), (1e-33, 1e-30), (1e-36, 1e-30)):
        x = g * norm
        want = definition(x, eps=eps)
        assert rel_err(GF.orthogonalize(x, eps=eps), want) < 1e-5, (norm, eps)
        mixed = torch.stack([g, x, torch.zeros_like(g), 3 * g])
        got = GF.orthogonalize(mixed, eps=eps)
        assert rel_err(got[1], want) < 1e-5 and torch.equal(got[2], torch.zeros_like(g))
    x = (g * 1e-13).bfloat16()
    assert rel_err(GF.orthogonalize(x), definition(x)) < 1e-5 + 2.0**-8
    for steps, coefficients in ((1, COEFFS), (8, COEFFS), (12, (1.5, -0.5, 0.0)), (3, (0.5, 0.1, 0.0))):
        # X is held under one power of two through all steps, so that what it grows to, by up to a factor a^steps, has room: at first
        # its norm then is as little as 1 / (2 a^steps), an entry of average size 1 / (2 a^steps sqrt(m n)), and an entry is held to
        # half of fp16's least step under the scale 2^14, 2^-25 / 2^14: 2^-38 a^steps sqrt(m n) relative to it.  (Eight steps of 512 x
        # 4608: 3.4445^8 = 19820, 1536 / 2^38 * 19820 = 1.1e-4, where 27 * 2^-22 alone is 6.4e-6.)
        faint = 2.0**-38 * max(1.0, coefficients[0]) ** steps * math.sqrt(m * n)
        want = definition(g * 1e-12, steps, coefficients)
        assert rel_err(GF.orthogonalize(g * 1e-12, steps=steps, coefficients=coefficients), want) < 3 * (steps + 1) * 2.0**-22 + faint, steps
    p, buf = torch.zeros_like(g), torch.zeros_like(g)
    muon_step([p], [g * 1e-12], [buf], lr=1.0, momentum=0.5, adjust_lr_fn="none")
    assert rel_err(-p, definition(g * 0.75e-12)) < 1e-5


@pytest.mark.gpu
def test_parameters_without_a_gradient_stay_out(dev):
    """Whose .grad is None is skipped in every step, not in the first one only: no decay, no update by what its momentum still
    holds (an orthogonalised momentum is full-sized however small it has become), the state as it was, .grad None as it was."""
    from torch import nn

    from gan_amd.optim import make_optimizer

    torch.manual_seed(4)
    net = nn.ModuleList([nn.Linear(12, 8), nn.Linear(8, 6), nn.Conv2d(2, 3, 3)]).to(dev)
    opt = make_optimizer("Muon", net, 0.05, {"weight_decay": 0.1})
    params = list(net.parameters())
    for p in params:
        p.grad = torch.randn_like(p)
    opt.step()  # momentum for all of them
    idle = params[2:4]
    held = [p.detach().clone() for p in idle]
    state = [{k: v.clone() for k, v in opt.state[p].items() if k != "step"} for p in idle]
    for p in idle:
        p.grad = None
    for _ in range(3):
        before = [p.detach().clone() for p in params]
        for p in params[:2] + params[4:]:
            p.grad = torch.randn_like(p)
        opt.step()
        for i, (p, q) in enumerate(zip(params, before)):
            assert torch.equal(p, q) == (i in (2, 3)), i
        assert all(p.grad is None for p in idle)
    for p, h, s in zip(idle, held, state):
        assert torch.equal(p, h) and all(torch.equal(opt.state[p][k], v) for k, v in s.items())
    for p in params:  # and they come back
        p.grad = torch.randn_like(p)
    opt.step()
    assert not any(torch.equal(p, h) for p, h in zip(idle, held))
