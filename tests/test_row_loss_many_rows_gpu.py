"""The row losses where every CTA, and every cluster of CTAs, goes through many rows, nearly all of them live: buffers that are used in turn,
rows fetched ahead, losses settled eight at a time, gradients over the logits.  Every row has labels and a gradient of its own, so that
a value of another row shows.  64-bit values are formed on the device, some rows at a time.

Tolerances: u = 2^-24.  An exponential exp((x - m) / T) is off by (3 |arg| + 3) u, |arg| averaged over the row under q; the row's sum adds a
rounding per level, ncol / 512 + 24 at most.  log q is off by that absolutely, plus 3 u per unit of the label's own argument."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SLICE = 1 << 24          # logits that are compared at once


def _soft(torch, x, temp):
    arg = (x.double() - x.double().amax(-1, keepdim=True)) / temp
    q = torch.exp(arg)
    s = q.sum(-1, keepdim=True)
    q = q / s
    rel = U * (3 * (q * arg.abs()).sum(-1, keepdim=True) + 3 + x.shape[1] / 512 + 24)
    return q, arg - torch.log(s), arg, rel


def _near(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist(), tol[bad][:4].tolist())


def _logits(torch, n, c, off, gen):
    """n rows of c logits that begin `off` floats behind a 16-byte boundary, and their own copy."""
    flat = torch.randn(off + n * c, device="cuda", generator=gen) * 2.5
    return flat, flat[off:].view(n, c), flat.data_ptr() + 4 * off


def _distill_check(torch, x, idx, t, temp, gy, y, gx):
    for rows in torch.arange(len(x), device="cuda").split(max(1, SLICE // x.shape[1])):
        q, logq, arg, rel = _soft(torch, x[rows], temp)
        used = idx[rows] >= 0
        at = idx[rows].long().clamp(min=0)
        live = used.any(-1)
        te = torch.where(used | ~live[:, None], t[rows].double() / temp, -torch.inf)
        parg = te - te.amax(-1, keepdim=True)
        p = torch.where(used, torch.softmax(te, -1), 0.0)
        parg = torch.where(used, parg, 0.0)
        logp = torch.where(p > 0, torch.log(torch.where(p > 0, p, 1.0)), 0.0)
        k = idx.shape[1]
        prel = U * (3 * (p * parg.abs()).sum(-1, keepdim=True) + 3 + k / 512 + 24)
        want = torch.where(live, temp ** 2 * (p * (logp - logq.gather(1, at))).sum(-1), 0.0)
        gap = parg.abs() + arg.gather(1, at).abs()
        tol = temp ** 2 * ((p * gap * ((3 * parg.abs() + 8) * U + prel)).sum(-1) + prel[:, 0] + rel[:, 0]) + 2 * U * want.abs()
        _near(y[rows], want, torch.where(live, tol, 0.0))
        w = torch.zeros_like(q).scatter_add_(1, at, p)
        ew = torch.zeros_like(q).scatter_add_(1, at, p * ((3 * parg.abs() + 4 + k) * U + prel))
        g = torch.where(live, gy[rows].double() * temp, 0.0)[:, None]
        _near(gx[rows], g * (q - w), g.abs() * (q * ((3 * arg.abs() + 8) * U + rel) + ew + 4 * U * w) + torch.where(live, 1e-38, 0.0)[:, None])


# Columns and what takes them: a CTA per row of 64 threads (many labels) and of 128, clusters of four CTAs and of eight.  Rows: more than
# eight for each CTA or cluster that fits the device, and no multiple of anything.
SHAPES = [(30011, 1000, 260), (9001, 8195, 20), (2503, 32003, 40), (403, 200003, 9)]


@pytest.mark.parametrize("over", [False, True])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("shape", SHAPES)
def test_distill(torch_cuda, vm, shape, mode, off, over):
    torch = torch_cuda
    n, c, k = shape
    gen = torch.Generator(device="cuda").manual_seed(n + off)
    flat, x, px = _logits(torch, n, c, off, gen)
    kept = x.clone()
    temp, ht = 1.5, torch.tensor([1.5], device="cuda")
    start = torch.randint(0, c, (n, 1), device="cuda", generator=gen)
    idx = ((start + torch.arange(k, device="cuda") * (c // k)) % c).int()
    idx[::5, 1] = idx[::5, 0]                                          # an id twice
    idx[torch.rand((n, k), device="cuda", generator=gen) < 0.1] = -1   # gaps
    idx[torch.rand(n, device="cuda", generator=gen) < 0.1] = -1        # padding rows
    t = torch.randn((n, k), device="cuda", generator=gen) * 3
    gy = torch.randn(n, device="cuda", generator=gen)
    y = torch.full((n,), float("nan"), device="cuda")
    gx = x if over else torch.full((n, c), float("nan"), device="cuda")
    pgx = px if over else gx
    if mode == "step":
        vm.softmax_top_distill_step(0, y, pgx, gy, px, idx, t, n, c, k, ht)
    else:
        ps = torch.empty((n, 3), device="cuda")
        vm.softmax_top_distill(0, y, ps, px, idx, t, n, c, k, ht)
        vm.softmax_top_distill_backward_x(0, pgx, gy, px, ps, idx, t, n, c, k, ht)
    torch.cuda.synchronize()
    _distill_check(torch, kept, idx, t, temp, gy, y, gx)


@pytest.mark.parametrize("over", [False, True])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("shape", SHAPES[1:])
def test_policy(torch_cuda, vm, shape, mode, off, over):
    torch = torch_cuda
    n, c, _ = shape
    gen = torch.Generator(device="cuda").manual_seed(n + off)
    flat, x, px = _logits(torch, n, c, off, gen)
    kept = x.clone()
    z = torch.randint(0, c, (n,), device="cuda", generator=gen)
    now = torch.cat([_soft(torch, x[r], 1.0)[1].gather(1, z[r][:, None])[:, 0]
                     for r in torch.arange(n, device="cuda").split(max(1, SLICE // c))])
    # ratios on both sides of the bounds 0.8 and 1.3, none next to them
    side = torch.tensor([0.5, 0.7, 0.9, 1.0, 1.1, 1.2, 1.5, 2.0], device="cuda").log()
    old = (now - side[torch.randint(0, 8, (n,), device="cuda", generator=gen)]).float()
    ref = (now + 0.4 * torch.randn(n, device="cuda", generator=gen)).float()
    adv, gy = (torch.randn(n, device="cuda", generator=gen) for _ in range(2))
    live = torch.rand(n, device="cuda", generator=gen) < 0.9
    pz = torch.where(live, z, -1).int()
    hypers = [torch.tensor([v], device="cuda") for v in (0.2, 0.3, 0.1)]
    y, logp = (torch.full((n,), float("nan"), device="cuda") for _ in range(2))
    gx = x if over else torch.full((n, c), float("nan"), device="cuda")
    pgx = px if over else gx
    if mode == "step":
        vm.softmax_policy_loss_step(0, y, logp, pgx, gy, px, pz, old, ref, adv, n, c, *hypers)
    else:
        ps = torch.empty((n, 3), device="cuda")
        vm.softmax_policy_loss(0, y, logp, ps, px, pz, old, ref, adv, n, c, *hypers)
        vm.softmax_policy_loss_backward_x(0, pgx, gy, px, ps, pz, n, c)
    torch.cuda.synchronize()
    for rows in torch.arange(n, device="cuda").split(max(1, SLICE // c)):
        on = live[rows]
        q, logq, arg, rel = _soft(torch, kept[rows], 1.0)
        l, a = (v.gather(1, z[rows][:, None])[:, 0] for v in (logq, arg))
        el = rel[:, 0] + 3 * U * a.abs()                              # error of l
        _near(logp[rows], torch.where(on, l, 0.0), torch.where(on, el + 2 * U * l.abs(), 0.0))
        av, dr = adv[rows].double(), ref[rows].double() - l
        rho = torch.exp(l - old[rows].double())
        er = rho * (el + 3 * U * (1 + (l - old[rows].double()).abs()))
        bound = rho.clamp(0.8, 1.3)
        free = rho * av <= bound * av
        em = torch.expm1(dr)
        want = -torch.where(free, rho * av, bound * av) + 0.1 * (em - dr)
        ed = el + 2 * U * dr.abs()
        tol = av.abs() * er + 6 * U * (rho * av).abs() + 0.1 * (em.abs() * ed + 4 * U * (em.abs() + dr.abs())) + 2 * U * want.abs()
        _near(y[rows], torch.where(on, want, 0.0), torch.where(on, tol, 0.0))
        slope = torch.where(free, -av * rho, 0.0) - 0.1 * em
        es = av.abs() * er * free + 4 * U * (av * rho).abs() + 0.1 * (torch.exp(dr) * ed + 6 * U * em.abs()) + 2 * U * slope.abs()
        g = gy[rows].double()
        hot = torch.zeros_like(q).scatter_(1, z[rows][:, None], 1.0)
        k = torch.where(on, g * slope, 0.0)[:, None]
        tol = torch.where(on, g.abs() * es, 0.0)[:, None] * (hot + q) + k.abs() * (q * ((3 * arg.abs() + 8) * U + rel) + 4 * U * hot)
        _near(gx[rows], k * (hot - q), tol + torch.where(on, 1e-38, 0.0)[:, None])
