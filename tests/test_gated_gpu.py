"""The gated linear layer against 64 bits.

Tolerance: a product's sum is off by eps = 2e-6 of the root of the sum of squares of its terms at most (Frobenius): the split
schemes drop 2^-21 of a product, a sum kept in tensor memory drifts by 7e-9 per value for at most 128 values (9e-7), and
fp32 sums of at most 8192 random terms are off by 1.6e-6.  h = act(g) u and the two inner gradients carry that error of g and u through
their derivatives, and round a few times (activations within 8 units in the last place)."""
import numpy as np
import pytest

from helpers import to_dev, to_host

pytestmark = pytest.mark.gpu
EPS, U = 2e-6, 2.0 ** -24

ACTS = ["none", "relu", "leaky", "sigmoid", "tanh", "gelu", "selu", "mish", "swish"]


def _act(torch, name, g, alpha=0.1):
    f = torch.nn.functional
    return {"none": lambda v: v, "relu": torch.relu, "leaky": lambda v: torch.where(v > 0, v, alpha * v),
            "sigmoid": torch.sigmoid, "tanh": torch.tanh, "gelu": f.gelu, "selu": f.selu, "mish": f.mish, "swish": f.silu}[name](g)


def _inputs(m, k, f, bias, seed):
    rng = np.random.default_rng(seed)
    s = lambda *shape: rng.standard_normal(shape).astype(np.float32)              # noqa: E731
    return dict(x=s(m, k), wg=(s(f, k) / np.sqrt(max(k, 1))).astype(np.float32), wu=(s(f, k) / np.sqrt(max(k, 1))).astype(np.float32),
                bg=s(f) if bias else None, bu=s(f) if bias else None, gh=s(m, f))


def _truth(torch, a, act):
    """Values and gradients in 64 bits, and for each the Frobenius error allowed to it."""
    d = {n: None if v is None else torch.from_numpy(v).cuda().double() for n, v in a.items()}
    x, wg, wu = (d[n].requires_grad_() for n in ("x", "wg", "wu"))
    g, u = x @ wg.T, x @ wu.T
    eg, eu = (x.detach() ** 2) @ (wg.detach() ** 2).T, (x.detach() ** 2) @ (wu.detach() ** 2).T
    if d["bg"] is not None:
        g, u = g + d["bg"], u + d["bu"]
    g.retain_grad()
    av = _act(torch, act, g)
    slope, = torch.autograd.grad(av.sum(), g, create_graph=True)
    curve = torch.autograd.grad(slope.sum(), g, retain_graph=True)[0] if slope.requires_grad else torch.zeros_like(g)
    h = av * u
    gx, gwg, gwu, gg, gu = torch.autograd.grad(h, (x, wg, wu, g, u), d["gh"])
    g, u, av, slope, curve, gh = (t.detach() for t in (g, u, av, slope, curve, d["gh"]))
    dg, du = EPS * eg.sqrt() + 2 * U * g.abs(), EPS * eu.sqrt() + 2 * U * u.abs()
    eh = slope.abs() * u.abs() * dg + av.abs() * du + 10 * U * (h.detach().abs() + u.abs())
    egg = gh.abs() * (slope.abs() * du + u.abs() * curve.abs() * dg + 16 * U * u.abs())
    egu = gh.abs() * (slope.abs() * dg + 16 * U * (av.abs() + 1))
    x, wg, wu = x.detach(), wg.detach(), wu.detach()
    n = lambda t: float(t.norm())                                                   # noqa: E731
    # a product's error: its own, and its inner gradient's passed on
    tx = EPS * n(((gg ** 2) @ (wg ** 2) + (gu ** 2) @ (wu ** 2)).sqrt()) + n(((egg ** 2) @ (wg ** 2) + (egu ** 2) @ (wu ** 2)).sqrt())
    tg = EPS * n(((gg.T ** 2) @ (x ** 2)).sqrt()) + n(((egg.T ** 2) @ (x ** 2)).sqrt())
    tu = EPS * n(((gu.T ** 2) @ (x ** 2)).sqrt()) + n(((egu.T ** 2) @ (x ** 2)).sqrt())
    vals = dict(h=h.detach(), g=g, u=u, gg=gg, gu=gu, gx=gx, gwg=gwg, gwu=gwu)
    tols = dict(h=n(eh), g=n(dg), u=n(du), gg=n(egg), gu=n(egu), gx=tx, gwg=tg, gwu=tu)
    return vals, tols


def _dev(torch, a):
    return {n: None if v is None else to_dev(torch, v) for n, v in a.items()}


def _new(torch, *shape):
    return torch.full(shape, float("nan"), device="cuda")


def _check(vals, tols, got):
    for n, t in got.items():
        err = float((t.double() - vals[n]).norm())
        assert err <= tols[n] + 1e-30, (n, err, tols[n], float(vals[n].norm()))


def _forward(torch, vm, d, m, k, f, act, save=True, alpha=None, stream=None):
    h = _new(torch, m, f)
    g, u = (_new(torch, m, f), _new(torch, m, f)) if save else (None, None)
    vm.gated_linear_forward(0, h, g, u, d["wg"], d["wu"], d["x"], d["bg"], d["bu"], f, m, k, act, alpha, stream)
    return h, g, u


SHAPES = [(1, 1, 1), (1, 64, 96), (1, 4096, 128), (1, 257, 65), (2, 512, 130), (3, 1028, 77), (4, 256, 8), (7, 100, 33),
          (8, 1024, 64), (15, 2052, 129), (16, 512, 512), (17, 512, 96), (33, 130, 70), (24, 68, 9), (25, 4100, 61),
          (32, 1028, 33), (41, 260, 500), (48, 1024, 200), (64, 4096, 64),
          (100, 96, 300), (129, 257, 255), (391, 512, 1365), (256, 512, 1024), (2048, 64, 64), (300, 1000, 700),
          (1024, 1024, 1024), (1153, 2048, 640), (5, 3, 4096), (640, 2056, 515), (300, 1000, 1100), (300, 1001, 1100),
          (1290, 520, 1030), (1280, 4104, 1024), (4104, 256, 520)]


@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(torch_cuda, vm, shape):
    torch = torch_cuda
    m, k, f = shape
    act = ACTS[(m + k + f) % len(ACTS)]
    a = _inputs(m, k, f, f % 2 == 1, m + k)
    vals, tols = _truth(torch, a, act)
    d = _dev(torch, a)
    alpha = torch.tensor([0.1], device="cuda")
    h, g, u = _forward(torch, vm, d, m, k, f, act, alpha=alpha)
    h2, _, _ = _forward(torch, vm, d, m, k, f, act, save=False, alpha=alpha)
    gx, gwg, gwu, gg, gu = _new(torch, m, k), _new(torch, f, k), _new(torch, f, k), _new(torch, m, f), _new(torch, m, f)
    vm.gated_linear_backward(0, gx, gwg, gwu, gg, gu, d["gh"], g, u, d["wg"], d["wu"], d["x"], f, m, k, act, alpha)
    torch.cuda.synchronize()
    _check(vals, tols, dict(h=h, g=g, u=u, gg=gg, gu=gu, gx=gx, gwg=gwg, gwu=gwu))
    assert torch.equal(h, h2)                    # saving the factors does not change the result


@pytest.mark.parametrize("path", ["warp", "planes", "raw"])
@pytest.mark.parametrize("shape", [(17, 33, 35), (49, 64, 32), (33, 131, 70), (60, 132, 70), (100, 96, 300), (129, 257, 255), (200, 300, 130), (700, 40, 48)])
def test_every_kernel_at_odd_sizes(torch_cuda, pkg, vm, shape, path):
    """The sizes at which the dispatch changes kernels, moved out of the way."""
    torch = torch_cuda
    m, k, f = shape
    a = _inputs(m, k, f, True, m)
    vals, tols = _truth(torch, a, "swish")
    d = _dev(torch, a)
    old = [pkg.load().kai_get_option(n) for n in (b"gated_tc_flops", b"gated_raw_rows")]
    pkg.capi.call("kai_set_option", b"gated_tc_flops", (1 << 62) if path == "warp" else 0)
    pkg.capi.call("kai_set_option", b"gated_raw_rows", (1 << 40) if path == "raw" else 0)
    try:
        h, g, u = _forward(torch, vm, d, m, k, f, "swish")
        h2, _, _ = _forward(torch, vm, d, m, k, f, "swish", save=False)
        gx, gwg, gwu = _new(torch, m, k), torch.ones((f, k), device="cuda"), torch.zeros((f, k), device="cuda")
        gg, gu = _new(torch, m, f), _new(torch, m, f)
        vm.gated_linear_backward(0, gx, gwg, gwu, gg, gu, d["gh"], g, u, d["wg"], d["wu"], d["x"], f, m, k, "swish", acc_w=True)
        torch.cuda.synchronize()
    finally:
        pkg.capi.call("kai_set_option", b"gated_tc_flops", old[0])
        pkg.capi.call("kai_set_option", b"gated_raw_rows", old[1])
    tols["gwg"] += 2 * U * float((vals["gwg"].abs() + 1).norm())        # the addition's rounding, and the subtraction's
    _check(vals, tols, dict(h=h, g=g, u=u, gg=gg, gu=gu, gx=gx, gwg=gwg - 1, gwu=gwu))
    assert torch.equal(h, h2)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(3, 64, 40), (40, 512, 72), (640, 1024, 512)])
def test_every_activation(torch_cuda, vm, act, shape):
    torch = torch_cuda
    m, k, f = shape
    a = _inputs(m, k, f, True, 9)
    vals, tols = _truth(torch, a, act)
    d = _dev(torch, a)
    alpha = torch.tensor([0.1], device="cuda")
    h, g, u = _forward(torch, vm, d, m, k, f, act, alpha=alpha)
    gx, gwg, gwu = _new(torch, m, k), _new(torch, f, k), _new(torch, f, k)
    gg, gu = g.clone(), u.clone()                # over the saved factors
    vm.gated_linear_backward(0, gx, gwg, gwu, gg, gu, d["gh"], gg, gu, d["wg"], d["wu"], d["x"], f, m, k, act, alpha)
    torch.cuda.synchronize()
    _check(vals, tols, dict(h=h, g=g, u=u, gg=gg, gu=gu, gx=gx, gwg=gwg, gwu=gwu))


@pytest.mark.parametrize("shape", [(5, 96, 33), (200, 300, 130), (1024, 512, 640)])
def test_accumulation_and_parts(torch_cuda, vm, shape):
    """+= for either gradient, one without the other, the inner gradients over the incoming one."""
    torch = torch_cuda
    m, k, f = shape
    a = _inputs(m, k, f, False, 4)
    vals, tols = _truth(torch, a, "swish")
    d = _dev(torch, a)
    _, g, u = _forward(torch, vm, d, m, k, f, "swish")
    plain = [_new(torch, m, k), _new(torch, f, k), _new(torch, f, k), _new(torch, m, f), _new(torch, m, f)]
    args = (d["gh"], g, u, d["wg"], d["wu"], d["x"], f, m, k, "swish")
    vm.gated_linear_backward(0, *plain, *args)
    gx, gwg, gwu = torch.ones((m, k), device="cuda"), torch.ones((f, k), device="cuda"), 2 * torch.ones((f, k), device="cuda")
    gg, gu = _new(torch, m, f), _new(torch, m, f)
    vm.gated_linear_backward(0, gx, gwg, gwu, gg, gu, *args, acc_x=True, acc_w=True)
    torch.cuda.synchronize()
    for got, one, base in ((gx, plain[0], 1.0), (gwg, plain[1], 1.0), (gwu, plain[2], 2.0)):
        # the same sums plus one addition (and, where dx is two products, another order): a few roundings of either term
        assert float((got - base - one).abs().max()) <= 16 * U * (float(one.abs().max()) + base)
    only_x = _new(torch, m, k)
    over = d["gh"].clone()
    vm.gated_linear_backward(0, only_x, None, None, over, gu, over, *args[1:])
    only_g, only_u = _new(torch, f, k), _new(torch, f, k)
    vm.gated_linear_backward(0, None, only_g, only_u, gg, gu, *args)
    torch.cuda.synchronize()
    assert torch.equal(over, plain[3])
    for got, one in ((only_x, plain[0]), (only_g, plain[1]), (only_u, plain[2])):
        assert torch.equal(got, one)
    _check(vals, tols, dict(gx=only_x, gwg=only_g, gwu=only_u))


def test_empty_extents(torch_cuda, vm):
    torch = torch_cuda
    w, x, h = torch.ones((4, 6), device="cuda"), torch.ones((3, 6), device="cuda"), torch.full((3, 4), 7.0, device="cuda")
    b = torch.full((4,), 2.0, device="cuda")
    vm.gated_linear_forward(0, h, None, None, w, w, x, None, None, 4, 0, 6, "swish")       # no rows
    torch.cuda.synchronize()
    assert bool((h == 7.0).all())
    vm.gated_linear_forward(0, h, None, None, None, None, None, b, b, 4, 3, 0, "relu")     # no inputs: the biases alone
    torch.cuda.synchronize()
    assert bool((h == 4.0).all())
    gwg, gwu, gx = torch.full((4, 6), 7.0, device="cuda"), torch.full((4, 6), 7.0, device="cuda"), torch.full((3, 6), 7.0, device="cuda")
    vm.gated_linear_backward(0, None, gwg, gwu, None, None, None, None, None, w, w, None, 4, 0, 6, "relu")   # no rows
    vm.gated_linear_backward(0, gx, None, None, None, None, None, None, None, None, None, x, 0, 3, 6, "relu")   # no outputs
    torch.cuda.synchronize()
    assert float(gwg.abs().max()) == 0 and float(gwu.abs().max()) == 0 and float(gx.abs().max()) == 0


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("shape", [(1, 512, 96), (9, 260, 40), (40, 512, 64), (300, 520, 264)])
def test_interior_pointers(torch_cuda, vm, shape, off):
    """Operands that begin off the 16-byte grid."""
    torch = torch_cuda
    m, k, f = shape
    a = _inputs(m, k, f, True, off)
    vals, tols = _truth(torch, a, "gelu")
    keep = []

    def shifted(v):
        t = torch.zeros(v.size + off, device="cuda")
        t[off:] = to_dev(torch, v).flatten()
        keep.append(t)
        return t.data_ptr() + 4 * off

    p = {n: shifted(v) for n, v in a.items()}
    outs = {n: torch.full((int(np.prod(s)) + off,), float("nan"), device="cuda")
            for n, s in dict(h=(m, f), g=(m, f), u=(m, f), gg=(m, f), gu=(m, f), gx=(m, k), gwg=(f, k), gwu=(f, k)).items()}
    at = {n: t.data_ptr() + 4 * off for n, t in outs.items()}
    vm.gated_linear_forward(0, at["h"], at["g"], at["u"], p["wg"], p["wu"], p["x"], p["bg"], p["bu"], f, m, k, "gelu")
    vm.gated_linear_backward(0, at["gx"], at["gwg"], at["gwu"], at["gg"], at["gu"], p["gh"], at["g"], at["u"], p["wg"], p["wu"],
                             p["x"], f, m, k, "gelu")
    torch.cuda.synchronize()
    _check(vals, tols, {n: t[off:].view(vals[n].shape) for n, t in outs.items()})
    assert all(bool(t[:off].isnan().all()) for t in outs.values())


def test_poisoned_rows_stay_theirs(torch_cuda, vm):
    """NaN and infinity in one row of x reach that row's outputs only."""
    torch = torch_cuda
    for m, k, f in ((6, 512, 64), (40, 512, 64), (700, 512, 256)):
        a = _inputs(m, k, f, False, 2)
        d = _dev(torch, a)
        clean = _forward(torch, vm, d, m, k, f, "swish")[0]
        d["x"][3, 5] = float("nan")
        d["x"][1, 7] = float("inf")
        got = _forward(torch, vm, d, m, k, f, "swish")[0]
        torch.cuda.synchronize()
        rows = [r for r in range(m) if r not in (1, 3)]
        assert torch.equal(got[rows], clean[rows])
        assert bool(got[3].isnan().all())
