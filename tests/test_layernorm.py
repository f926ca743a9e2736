"""functional.layer_norm / modelling.common.LayerNorm: forward, backward and second order against the formulas in 64 bits.

Bounds are elementwise and counted in roundings of 2^-24 (plus half a step of bf16 where the result is one, 2^-8 of the value),
on the sum of the magnitudes that enter the value: a row sum is a tree over at most 32 additions in a thread, 6 in a wave,
16 over waves and 64 over pieces, under 128 roundings; every result is a product of at most three quantities that carry
one such sum each, so 512 roundings cover it."""
import pytest
import torch

U = 2.0**-24
N = 512


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def make(rows, d, dt, dev, seed=0, offset=0, mean=1.0):
    gen = torch.Generator(device="cpu").manual_seed(seed + 7 * rows + d)

    def t(scale=1.0, shift=0.0):
        flat = torch.randn(rows * d + offset, generator=gen) * scale + shift
        return flat.to(dt).to(dev)[offset:].view(rows, d)  # offset: rows that start between 16-byte boundaries

    x, g, v = t(1.5, mean), t(), t()
    w, b, cw, cb = (torch.randn(d, generator=gen).to(dev) for _ in range(4))
    return x, g, v, 1 + 0.2 * w, 0.2 * b, cw, cb


def proj(u, t):
    return u - u.mean(1, keepdim=True) - t * (u * t).mean(1, keepdim=True)


def proj_mag(u, t):
    u = u.abs()
    return u + u.mean(1, keepdim=True) + t.abs() * (u * t.abs()).mean(1, keepdim=True)


class Ref:
    """Every result in 64 bits, and beside it the magnitudes that its roundings go by."""

    def __init__(self, x, g, v, w, b, cw=None, cb=None, eps=1e-5):
        x, g, v, w, b = (t.detach().double() for t in (x, g, v, w, b))
        cw = torch.zeros_like(w) if cw is None else cw.double()
        cb = torch.zeros_like(w) if cb is None else cb.double()
        m = x.mean(1, keepdim=True)
        r = ((x - m).square().mean(1, keepdim=True) + eps).rsqrt()
        t = (x - m) * r
        ta = t.abs() + (x.abs().mean(1, keepdim=True) + x.abs()) * r  # t and what the rounding of its mean and difference adds
        h = g * w
        self.y, self.y_mag = t * w + b, ta * w.abs() + b.abs()
        self.gx, self.gx_mag = r * proj(h, t), r * proj_mag(h, ta)
        self.gw, self.gw_mag = (g * t).sum(0), (g.abs() * ta).sum(0)
        self.gb, self.gb_mag = g.sum(0), g.abs().sum(0)
        pv, pv_mag = r * proj(v, t), r * proj_mag(v, ta)
        self.gg, self.gg_mag = w * pv + cw * t + cb, w.abs() * pv_mag + cw.abs() * ta + cb.abs()
        self.gww, self.gww_mag = (g * pv).sum(0), (g.abs() * pv_mag).sum(0)
        ht, vt = (h * t).mean(1, keepdim=True), (v * t).mean(1, keepdim=True)
        hta, vta = (h.abs() * ta).mean(1, keepdim=True), (v.abs() * ta).mean(1, keepdim=True)
        s = (v * h).mean(1, keepdim=True) - v.mean(1, keepdim=True) * h.mean(1, keepdim=True) - vt * ht
        sa = (v * h).abs().mean(1, keepdim=True) + v.abs().mean(1, keepdim=True) * h.abs().mean(1, keepdim=True) + vta * hta
        self.gxx = r * proj(g * cw - r * (v * ht + h * vt), t) - r.square() * t * s
        self.gxx_mag = r * proj_mag((g * cw).abs() + r * (v.abs() * hta + h.abs() * vta), ta) + r.square() * ta * sa


def near(got, ref, name, rows=0):
    want, mag = getattr(ref, name), getattr(ref, name + "_mag")
    assert got.shape == want.shape
    lim = (N + rows) * U * mag + (2.0**-8 * want.abs() if got.dtype == torch.bfloat16 else 0) + 1e-37
    off = (got.detach().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= lim).all(), (name, float((off / lim).max()))


# (rows, width): one element, tails, each number of threads a row, both ways of summing columns, pieces of long rows
SHAPES = [
    (1, 1), (3, 2), (5, 7), (1, 16), (32, 128), (7, 1000), (4099, 33), (2051, 64), (1300, 257), (1100, 1500), (1030, 3001),
    (1026, 8000), (600, 513), (65, 4096), (3, 8192), (130, 12000), (3, 16384), (2, 16387), (5, 33001), (1, 100003), (70, 66000),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d", SHAPES)
def test_three_orders(dev, rows, d, dt):
    from gan_amd import functional as GF

    x, g, v, w, b, _, _ = make(rows, d, dt, dev)
    ref = Ref(x, g, v, w, b)
    x.requires_grad_(), g.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = GF.layer_norm(x, d, w, b)
    near(y, ref, "y")
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g.detach(), retain_graph=True)
    assert gx.dtype == dt and gw.dtype == gb.dtype == torch.float32
    near(gx, ref, "gx")
    near(gw, ref, "gw", rows)
    near(gb, ref, "gb", rows)
    (gx,) = torch.autograd.grad(y, x, g, create_graph=True)
    near(gx, ref, "gx")
    gxx, gg, gww = torch.autograd.grad(gx, (x, g, w), v)
    near(gxx, ref, "gxx")
    near(gg, ref, "gg")
    near(gww, ref, "gww", rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d", [(40, 300), (1030, 260), (6, 20000), (3, 70000)])
def test_second_order_of_all_three_gradients(dev, rows, d, dt):
    """A loss that takes gx, gw and gb again: cotangents for all of them."""
    from gan_amd import functional as GF

    x, g, v, w, b, cw, cb = make(rows, d, dt, dev)
    ref = Ref(x, g, v, w, b, cw, cb)
    x.requires_grad_(), g.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = GF.layer_norm(x, d, w, b)
    outs = torch.autograd.grad(y, (x, w, b), g, create_graph=True)
    gxx, gg, gww = torch.autograd.grad(outs, (x, g, w), (v, cw, cb))
    near(gxx, ref, "gxx")
    near(gg, ref, "gg")
    near(gww, ref, "gww", rows)
    # only the weight's gradient taken again
    zero = torch.zeros_like(v)
    ref = Ref(x, g, zero, w, b, cw)
    (gw,) = torch.autograd.grad(GF.layer_norm(x, d, w, b), w, g, create_graph=True)
    gxx, gg = torch.autograd.grad(gw, (x, g), cw)
    near(gxx, ref, "gxx")
    near(gg, ref, "gg")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_off_boundary_rows_and_no_affine(dev, dt):
    from gan_amd import functional as GF

    for rows, d, offset in ((9, 1000, 1), (1050, 64, 3), (4, 18000, 1), (3, 5, 2)):
        x, g, v, w, b, _, _ = make(rows, d, dt, dev, offset=offset)
        assert x.data_ptr() % 16 and x.is_contiguous()
        ones, zeros = torch.ones_like(w), torch.zeros_like(b)
        for w_, b_ in ((w, b), (None, None), (w, None), (None, b)):
            ref = Ref(x, g, v, ones if w_ is None else w_, zeros if b_ is None else b_)
            xr, gr = x.detach().requires_grad_(), g.detach().requires_grad_()
            y = GF.layer_norm(xr, (d,), w_, b_)
            near(y, ref, "y")
            (gx,) = torch.autograd.grad(y, xr, gr, create_graph=True)
            near(gx, ref, "gx")
            gxx, gg = torch.autograd.grad(gx, (xr, gr), v)
            near(gxx, ref, "gxx")
            near(gg, ref, "gg")


@pytest.mark.gpu
def test_layouts_and_parameter_types(dev):
    from gan_amd import functional as GF
    from gan_amd.modelling.common import LayerNorm

    torch.manual_seed(3)
    # whole samples of a channels-last activation, read as it lies
    x = torch.randn(6, 24, 5, 7, device=dev).contiguous(memory_format=torch.channels_last).requires_grad_()
    norm = LayerNorm((24, 5, 7)).to(dev)
    with torch.no_grad():
        norm.weight.normal_(1, 0.2), norm.bias.normal_(0, 0.2)
    y = norm(x)
    assert y.is_contiguous(memory_format=torch.channels_last)
    g = torch.randn_like(x)
    ref = Ref(x.reshape(6, -1), g.reshape(6, -1), g.reshape(6, -1), norm.weight.reshape(-1), norm.bias.reshape(-1))
    near(y.reshape(6, -1), ref, "y")
    gx, gw, gb = torch.autograd.grad(y, (x, norm.weight, norm.bias), g, create_graph=True)
    near(gx.reshape(6, -1), ref, "gx")
    near(gw.reshape(-1), ref, "gw", 6)
    near(gb.reshape(-1), ref, "gb", 6)
    gxx, gww = torch.autograd.grad(gx, (x, norm.weight), g)
    near(gxx.reshape(6, -1), ref, "gxx")
    near(gww.reshape(-1), ref, "gww", 6)
    # strided input, bfloat16 parameters, five dimensions, autocast
    wide = torch.randn(4, 3, 2, 5, 48, device=dev)[..., ::2]
    w, b = torch.randn(5, 24, device=dev).bfloat16(), torch.randn(5, 24, device=dev).bfloat16()
    ref = Ref(wide.reshape(24, 120), wide.reshape(24, 120), wide.reshape(24, 120), w.reshape(-1), b.reshape(-1))
    wr = w.requires_grad_()
    y = GF.layer_norm(wide, (5, 24), wr, b)
    near(y.reshape(24, 120), ref, "y")
    (gw,) = torch.autograd.grad(y, wr, wide.contiguous())
    assert gw.dtype == torch.bfloat16 and gw.shape == w.shape
    near(gw.reshape(-1), ref, "gw", 24)
    norm = LayerNorm(32).to(dev)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert norm(torch.randn(5, 32, device=dev)).dtype == torch.bfloat16
    # nothing to normalise
    e = torch.empty(0, 8, device=dev, requires_grad=True)
    w0 = torch.ones(8, device=dev, requires_grad=True)
    y = GF.layer_norm(e, 8, w0)
    ge, gw = torch.autograd.grad(y.sum(), (e, w0))
    assert y.shape == ge.shape == (0, 8) and torch.equal(gw, torch.zeros(8, device=dev))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [24, 700, 5000, 40000])
def test_rows_do_not_touch_each_other(dev, d):
    """A row of NaN, of infinities, of one value, and of the largest finite numbers' scale: the others keep their bits."""
    from gan_amd import functional as GF

    x, g, v, w, b, _, _ = make(9, d, torch.float32, dev)
    clean_x = x.clone()
    bad = x.clone()
    bad[2] = float("nan")
    bad[4, d // 2] = float("inf")
    bad[6] = 3.25
    keep = [i for i in range(9) if i not in (2, 4, 6)]

    def all_three(x):
        xr, gr = x.clone().requires_grad_(), g.clone().requires_grad_()
        y = GF.layer_norm(xr, d, w, b)
        (gx,) = torch.autograd.grad(y, xr, gr, create_graph=True)
        return (y, gx, *torch.autograd.grad(gx, (xr, gr), v))

    a, c = all_three(bad), all_three(clean_x)
    for p, q in zip(a, c):
        assert torch.equal(p[keep], q[keep])
        assert torch.isnan(p[2]).all() and torch.isfinite(p[6]).all()
    assert torch.equal(a[0][6], b)  # (x - mean is zero)
    far = make(5, d, torch.float32, dev, mean=1000.0)  # a mean far from zero: the variance is that of the differences
    near(GF.layer_norm(far[0], d, far[3], far[4]), Ref(*far[:5]), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", [(6, 40), (3, 20000)])
def test_gradients_against_differences(dev, rows, d):
    """Central differences of the kernels' own outputs along a random direction.  With a step of 2^-6 of x's spread the third
    derivative leaves about 2^-12 of the slope; rounding leaves 2^-24 of the summed magnitudes over the step, summed in 64
    bits over outputs of random sign: under 2^-24 * 2^6 * sqrt(outputs) against a slope of about sqrt(outputs)."""
    from gan_amd import functional as GF

    x, g, v, w, b, _, _ = make(rows, d, torch.float32, dev, mean=0.3)
    gen = torch.Generator(device="cpu").manual_seed(5)
    step = torch.randn(rows, d, generator=gen).to(dev)
    eps = 2.0**-6

    def first(x):
        return (GF.layer_norm(x, d, w, b).double() * g.double()).sum()

    def slope_of(x):
        xr = x.clone().requires_grad_()
        return torch.autograd.grad(GF.layer_norm(xr, d, w, b), xr, g)[0]

    def second(x):
        return (slope_of(x).double() * v.double()).sum()

    xr, gr = x.clone().requires_grad_(), g.clone().requires_grad_()
    (gx,) = torch.autograd.grad(GF.layer_norm(xr, d, w, b), xr, gr, create_graph=True)
    (gxx,) = torch.autograd.grad(gx, xr, v)
    scale = (rows * d) ** 0.5
    for f, grad in ((first, gx), (second, gxx)):
        num = (f(x + eps * step) - f(x - eps * step)) / (2 * eps)
        assert abs(float(num) - float((grad.double() * step.double()).sum())) <= 2.0**-9 * scale


@pytest.mark.gpu
def test_same_bits_other_stream_and_graph(dev):
    from gan_amd import functional as GF

    cases = [make(1200, 300, torch.bfloat16, dev), make(20, 9000, torch.float32, dev), make(4, 50000, torch.float32, dev)]

    def step():
        out = []
        for x, g, v, w, b, _, _ in cases:
            xr, gr, wr, br = (t.detach().requires_grad_() for t in (x, g, w, b))
            y = GF.layer_norm(xr, x.shape[1], wr, br)
            out += [y, *torch.autograd.grad(y, (wr, br), g, retain_graph=True)]
            (gx,) = torch.autograd.grad(y, xr, gr, create_graph=True)
            out += [gx, *torch.autograd.grad(gx, (xr, gr, wr), v)]
        return [t.detach() for t in out]

    want = [t.clone() for t in step()]
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        for x, g, v, *_ in cases:  # new numbers in the same places
            x.copy_(x.flip(0)), g.mul_(-1), v.copy_(v.flip(0))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, held)), k


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d", [(1, 1), (5, 24), (3, 700), (4, 5000), (2, 40000)])
def test_without_gradients(dev, rows, d, dt):
    """Where nothing asks for a gradient the same bits come back and nothing is kept."""
    from gan_amd import functional as GF

    torch.manual_seed(rows + d)
    x = torch.randn(rows, d, device=dev).to(dt)
    w, b = torch.randn(d, device=dev, requires_grad=True), torch.randn(d, device=dev, requires_grad=True)
    want = GF.layer_norm(x, d, w, b)
    assert want.requires_grad
    with torch.no_grad():
        got = GF.layer_norm(x, d, w, b)
    assert not got.requires_grad and torch.equal(got, want)
    assert torch.equal(GF.layer_norm(x, d, w.detach(), b.detach()), want)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
        GF.layer_norm(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), d, w.detach())


@pytest.mark.gpu
def test_third_order_is_refused(dev):
    from gan_amd import functional as GF

    x = torch.randn(4, 8, device=dev, requires_grad=True)
    y = GF.layer_norm(x, 8)
    (g1,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    (g2,) = torch.autograd.grad(g1.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g2.sum().backward()


def test_refusals():
    from gan_amd import _lib
    from gan_amd import functional as GF

    x = torch.randn(4, 8)
    for kw in (
        dict(normalized_shape=8),  # not on a ROCm device
        dict(normalized_shape=7),
        dict(normalized_shape=()),
        dict(normalized_shape=(2, 4, 8)),
        dict(normalized_shape=0),
        dict(normalized_shape=8, weight=torch.ones(4)),
        dict(normalized_shape=8, weight=torch.ones(8, dtype=torch.int32)),
        dict(normalized_shape=8, bias=torch.ones(1, 8)),
        dict(normalized_shape=8, eps=-1.0),
        dict(normalized_shape=8, eps=float("nan")),
    ):
        with pytest.raises(_lib.GanAmdError):
            GF.layer_norm(x, **kw)
    with pytest.raises(_lib.GanAmdError):
        GF.layer_norm(x.half(), 8)
    # the C entries refuse before anything is launched
    lib = _lib.load()
    p = 4096  # never read
    assert lib.gan_layernorm_workspace(-1, 8, 0, 0, 0) < 0 and lib.gan_layernorm_workspace(1, 0, 0, 0, 0) < 0
    assert lib.gan_layernorm_workspace(1, 8, 2, 0, 0) < 0 and lib.gan_layernorm_workspace(1, 8, 0, 3, 0) < 0
    assert lib.gan_layernorm_workspace(0, 8, 0, 1, 1) == 0
    assert lib.gan_layernorm_fwd(None, p, p, p, p, 4, 8, 1e-5, 0, None, 0, None) != 0
    assert lib.gan_layernorm_fwd(p, p, p, p, p, 4, 0, 1e-5, 0, None, 0, None) != 0
    assert lib.gan_layernorm_fwd(p, p, p, p, p, 4, 8, -1.0, 0, None, 0, None) != 0
    assert lib.gan_layernorm_fwd(p, p, p, p, p + 4, 4, 8, 1e-5, 0, None, 0, None) != 0
    assert lib.gan_layernorm_fwd(p, p, p, p, p, 4, 8, 1e-5, 7, None, 0, None) != 0
    assert lib.gan_layernorm_fwd(p, p, p, p, p, 1 << 31, 8, 1e-5, 0, None, 0, None) != 0
    need = lib.gan_layernorm_workspace(4, 1 << 20, 0, 0, 0)
    assert need > 0 and lib.gan_layernorm_fwd(p, p, p, p, p, 4, 1 << 20, 1e-5, 0, p, need - 1, None) != 0
    assert b"workspace" in lib.gan_amd_last_error()
    assert lib.gan_layernorm_bwd(p, p, p, None, p, p, 4, 8, 0, p, 1 << 20, None) != 0
    assert lib.gan_layernorm_bwd(p, p, p, p, p, p, 0, 8, 0, p, 1 << 20, None) != 0
    assert lib.gan_layernorm_bwd2(None, p, p, p, p, p, p, p, p, p, 4, 8, 0, p, 1 << 20, None) != 0
    assert lib.gan_layernorm_bwd2(p, p, p, p, p, p, p, p, p, p, 4, 8, 0, p + 4, 1 << 20, None) != 0


def plain_launches(monkeypatch):
    """The three launches as their formulas on the CPU: what lies between them and the engine is then what is tested."""
    from gan_amd import functional as GF

    def t_of(x, stats, d):
        x, stats = x.detach().reshape(-1, d).double(), stats.double()
        return (x - stats[:, :1]) * stats[:, 1:]

    def fwd(x, weight, bias, d, eps, keep=True):
        u = x.detach().reshape(-1, d).double()
        m = u.mean(1, keepdim=True)
        stats = torch.cat([m, ((u - m).square().mean(1, keepdim=True) + eps).rsqrt()], 1)
        y = (u - m) * stats[:, 1:]
        y = y if weight is None else y * weight.detach().reshape(d).double()
        y = y if bias is None else y + bias.detach().reshape(d).double()
        return y.to(x.dtype).view(x.shape), stats.float()

    def bwd(g, x, weight, stats, d, need_x, need_cols):
        t, u, r = t_of(x, stats, d), g.detach().reshape(-1, d).double(), stats[:, 1:].double()
        h = u if weight is None else u * weight.detach().reshape(d).double()
        gx = torch.empty_like(x).copy_((r * proj(h, t)).view(x.shape)) if need_x else None
        return gx, torch.stack([(u * t).sum(0), u.sum(0)]).float() if need_cols else None

    def bwd2(v, cw, cb, g, x, weight, stats, d, need_g, need_x, need_w):
        flat = [s.detach().reshape(-1, d) for s in (x, g, v)]
        one = torch.ones(d, dtype=torch.float64)
        w = one if weight is None else weight.detach().reshape(d)
        ref = Ref(*flat, w, one, *(None if s is None else s.detach().reshape(d) for s in (cw, cb)))
        gg, gxx = (torch.empty_like(x).copy_(getattr(ref, k).view(x.shape)) if need else None for k, need in (("gg", need_g), ("gxx", need_x)))
        return gg, gxx, ref.gww.float() if need_w else None

    monkeypatch.setattr(GF, "raw_layer_norm", fwd)
    monkeypatch.setattr(GF, "raw_layer_norm_bwd", bwd)
    monkeypatch.setattr(GF, "raw_layer_norm_bwd2", bwd2)


def check_gradients_asked_for_alone(norm, dev, has_weight):
    """Under create_graph, any of the gradients without the others (whose tensors require one all the same)."""
    rows, d = 12, 40
    x0, g0, v, w0, b0, cw, cb = make(rows, d, torch.float32, dev)
    one, zero = torch.ones_like(w0), torch.zeros_like(w0)
    for asked in ("x", "w", "b", "xw", "xb", "wb", "xwb"):
        if "w" in asked and not has_weight:
            continue
        leaf = dict(zip("xgwb", (t.clone().requires_grad_() for t in (x0, g0, w0, b0))))
        w = leaf["w"] if has_weight else None
        ref = Ref(x0, g0, v if "x" in asked else torch.zeros_like(v), w0 if has_weight else one, b0, cw if "w" in asked else zero, cb if "b" in asked else zero)
        got = dict(zip(asked, torch.autograd.grad(norm(leaf["x"], w, leaf["b"]), [leaf[k] for k in asked], leaf["g"], create_graph=True)))
        for k in asked:
            near(got[k], Ref(x0, g0, v, w0 if has_weight else one, b0), "g" + k, rows)
        (gg,) = torch.autograd.grad([got[k] for k in asked], leaf["g"], [{"x": v, "w": cw, "b": cb}[k] for k in asked])
        near(gg, ref, "gg")
    # handed to backward() by name
    x, w, b = (t.clone().requires_grad_() for t in (x0, w0, b0))
    norm(x, w if has_weight else None, b).backward(g0, inputs=[b], create_graph=True)
    near(b.grad.detach(), Ref(x0, g0, v, w0 if has_weight else one, b0), "gb", rows)
    assert x.grad is None and w.grad is None
    b.grad = None  # (else it and its graph hold each other)
    # a bias computed from what the gradient is taken of
    c = b0.clone().requires_grad_()
    y = norm(x, w if has_weight else None, 0.5 * c)
    (gc,) = torch.autograd.grad([y, c], c, [g0, torch.ones_like(c)], create_graph=True)
    near((gc.detach() - 1) * 2, Ref(x0, g0, v, w0, b0), "gb", rows + N)  # (1 is added and taken off: another rounding of 1 + |gb|)


@pytest.mark.parametrize("has_weight", [True, False])
def test_gradients_asked_for_alone(monkeypatch, has_weight):
    from gan_amd import functional as GF

    plain_launches(monkeypatch)
    check_gradients_asked_for_alone(lambda x, w, b: GF.LayerNormFn.apply(x, w, b, 40, 1e-5), torch.device("cpu"), has_weight)


@pytest.mark.gpu
@pytest.mark.parametrize("has_weight", [True, False])
def test_gradients_asked_for_alone_on_the_device(dev, has_weight):
    from gan_amd import functional as GF

    check_gradients_asked_for_alone(lambda x, w, b: GF.layer_norm(x, 40, w, b), dev, has_weight)

    def samples(x, w, b):  # whole samples of a channels-last activation
        x = x.view(12, 2, 5, 4).permute(0, 3, 1, 2)
        w, b = (None if t is None else t.view(2, 5, 4).permute(2, 0, 1) for t in (w, b))
        return GF.layer_norm(x, (4, 2, 5), w, b).permute(0, 2, 3, 1).reshape(12, 40)

    check_gradients_asked_for_alone(samples, dev, has_weight)


def check_gradients_changed_in_place(norm, dev):
    """The gradients are tensors of their own, as F.layer_norm's are: each may be scaled or clipped where it lies."""
    rows, d = 6, 40
    x0, g0, _, w0, b0, cw, cb = make(rows, d, torch.float32, dev)
    ref = Ref(x0, g0, torch.zeros_like(x0), w0, b0, 2 * cw, 3 * cb)
    x, g, w, b = (t.clone().requires_grad_() for t in (x0, g0, w0, b0))
    gw, gb = torch.autograd.grad(norm(x, w, b), (w, b), g, create_graph=True)
    gw.mul_(2), gb.mul_(3)
    near(gw.detach() / 2, ref, "gw", rows)
    near(gb.detach() / 3, ref, "gb", rows)
    near(torch.autograd.grad((gw, gb), g, (cw, cb))[0], ref, "gg")
    # those of a first and of a second backward without create_graph, by a factor that asks for a gradient itself
    factor = torch.full((), 2.0, device=dev, requires_grad=True)
    first = torch.autograd.grad(norm(x, w, b), (x, w, b), g0)
    (gx,) = torch.autograd.grad(norm(x, w, b), x, g, create_graph=True)
    for grad in (*first, *torch.autograd.grad(gx, (x, g, w), g0)):
        want = 2 * grad
        grad.mul_(factor)
        assert torch.equal(grad, want) and grad.requires_grad


def test_gradients_changed_in_place(monkeypatch):
    from gan_amd import functional as GF

    plain_launches(monkeypatch)
    dev = torch.device("cpu")
    check_gradients_changed_in_place(lambda x, w, b: GF.LayerNormFn.apply(x, w, b, 40, 1e-5), dev)
    shape = (4, 10)  # parameters of more than one dimension
    x, w, b = (t.requires_grad_() for t in (torch.randn(3, *shape), torch.randn(shape), torch.randn(shape)))
    factor = torch.full((), 2.0, requires_grad=True)
    for create_graph in (True, False):
        for grad in torch.autograd.grad(GF.LayerNormFn.apply(x, w, b, 40, 1e-5), (w, b), torch.randn(3, *shape), create_graph=create_graph):
            want = 2 * grad.detach()
            grad.mul_(factor)
            assert torch.equal(grad, want) and grad.shape == shape


@pytest.mark.gpu
def test_gradients_changed_in_place_on_the_device(dev):
    from gan_amd import functional as GF

    check_gradients_changed_in_place(lambda x, w, b: GF.layer_norm(x, 40, w, b), dev)


def test_workspace_query_refuses_what_the_calls_refuse():
    from gan_amd import _lib

    lib = _lib.load()
    p = 4096  # never read
    for rows, d, dtype in ((1 << 31, 8, 1), (1 << 62, 8, 1), (1 << 25, 1 << 15, 0), (64, 1 << 30, 0), (128, 1 << 30, 1), (1, (1 << 30) + 1, 0)):
        for order in range(3):
            assert lib.gan_layernorm_workspace(rows, d, dtype, order, 1) < 0, (rows, d, order)
        assert lib.gan_layernorm_fwd(p, p, p, p, p, rows, d, 1e-5, dtype, p, 1 << 62, None) != 0
        assert lib.gan_layernorm_bwd(p, p, p, p, p, p, rows, d, dtype, p, 1 << 62, None) != 0
        assert lib.gan_layernorm_bwd2(p, p, p, p, p, p, p, p, p, p, rows, d, dtype, p, 1 << 62, None) != 0
    for rows, d, dtype in (((1 << 31) - 1, 8, 1), (63, 1 << 30, 0), (1, 1 << 30, 0), (4096, 1 << 15, 0)):
        for order in range(3):
            assert lib.gan_layernorm_workspace(rows, d, dtype, order, 1) >= 0, (rows, d, order)


@pytest.mark.gpu
def test_the_longest_row(dev):
    """2^30 elements, a tail of 2^30 - 3, in fp32: the most tiles of columns and pieces of a row.  Sums go over 2^18 pieces here,
    1024 one after another in a thread: 1100 roundings, at most three such sums in a value, 4096 roundings asked."""
    from gan_amd import functional as GF

    for d in ((1 << 30) - 3, 1 << 30):
        torch.manual_seed(7)
        x = torch.randn(1, d, device=dev).add_(0.5).requires_grad_()
        w = torch.randn(d, device=dev).requires_grad_()
        b = torch.zeros(d, device=dev).requires_grad_()
        g = torch.randn(1, d, device=dev)
        y = GF.layer_norm(x, d, w, b)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
        parts = [slice(k, min(k + (1 << 27), d)) for k in range(0, d, 1 << 27)]
        x, w, g, y, gx = (t.detach().view(-1) for t in (x, w, g, y, gx))
        mean = sum(x[p].double().sum() for p in parts) / d
        size = sum(x[p].double().abs().sum() for p in parts) / d
        r = (sum((x[p].double() - mean).square().sum() for p in parts) / d + 1e-5).rsqrt()
        hm = sum((g[p].double() * w[p].double()).sum() for p in parts) / d
        ht = sum((g[p].double() * w[p].double() * (x[p].double() - mean) * r).sum() for p in parts) / d
        ha = sum((g[p].double() * w[p].double()).abs().sum() for p in parts) / d
        for p in (parts[0], parts[-1]):
            t = (x[p].double() - mean) * r
            ta = t.abs() + (size + x[p].double().abs()) * r
            h = g[p].double() * w[p].double()
            lim = 4096 * U
            assert ((y[p].double() - t * w[p].double()).abs() <= lim * ta * w[p].double().abs() + 1e-37).all()
            assert ((gw[p].double() - g[p].double() * t).abs() <= lim * g[p].double().abs() * ta + 1e-37).all()
            assert torch.equal(gb[p], g[p])
            # (|mean(h t)| <= mean |h| * max |t| and |t| < 8 here)
            assert ((gx[p].double() - r * (h - hm - t * ht)).abs() <= lim * r * (h.abs() + ha + 8 * ta * ha)).all()
        del x, w, b, g, y, gx, gw, gb, t, ta, h
        torch.cuda.empty_cache()
