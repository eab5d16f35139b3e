"""Losses on rows of logits (distillation from a teacher's top logits, clipped policy loss) against the definitions in
64 bits.

Tolerances.  u = 2^-24 is the relative error of one fp32 rounding.  An exponential exp((x - m) / T) is off by (3 |arg| + 3) u
(difference, factor, 1 / T; expf within an ulp and its own rounding), with |arg| averaged over the row under q; a sum over the row adds one
rounding per level, at most 4 * ncol / (4 * 512) + 24 levels here.  log q is then off by that much absolutely, plus u per unit of the
label's own argument.  Teacher probabilities likewise, over ntop entries."""

import numpy as np
import pytest

from helpers import to_dev, to_host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NAN = float("nan")


def _soft(x, temp):
    """q, log q, and the relative error allowed to the row's sum of exponentials."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        top = x.max(-1, keepdims=True)
        arg = (x - top) / temp
        e = np.exp(arg)
        s = e.sum(-1, keepdims=True)
        q = e / s
        mean = np.where(q > 0, q * np.abs(np.where(q > 0, arg, 0)), 0).sum(-1, keepdims=True)
        rel = U * (3 * mean + 3 + x.shape[-1] / 512 + 24)
        # where there is no probability there is no argument either: the value is 0 on both sides
        return q, arg - np.log(s), np.where(q > 0, arg, 0), rel


def _distill_truth(x, idx, t, temp, gy):
    n, c = x.shape
    y, gx, ty, tg = np.zeros(n), np.zeros((n, c)), np.zeros(n), np.zeros((n, c))
    q, logq, arg, rel = _soft(x, temp)
    for r in range(n):
        on = (idx[r] >= 0) & (t[r] > -np.inf)
        if not on.any():
            continue
        ids = idx[r][on]
        p, logp, parg, prel = _soft(t[r][on][None], temp)
        p, logp, parg, prel = p[0], logp[0], parg[0], float(prel[0, 0])
        y[r] = temp ** 2 * (p * (logp - logq[r, ids])).sum()
        # p is off by (3 |parg| + 4) u + prel, which multiplies the term; the logarithms by their sums' errors
        gap = np.abs(parg) + np.abs(arg[r, ids])
        ty[r] = temp ** 2 * ((p * gap * ((3 * np.abs(parg) + 8) * U + prel)).sum() + prel + float(rel[r, 0])) + 2 * U * abs(y[r])
        w = np.zeros(c)
        np.add.at(w, ids, p)
        ew = np.zeros(c)
        np.add.at(ew, ids, p * ((3 * np.abs(parg) + 4 + len(ids)) * U + prel))
        gx[r] = gy[r] * temp * (q[r] - w)
        tg[r] = abs(gy[r]) * temp * (q[r] * ((3 * np.abs(arg[r]) + 8) * U + rel[r]) + ew + 4 * U * w) + 1e-38
    return y, gx, ty, tg


def _table(rng, n, c, k, repeat=False):
    idx = np.stack([rng.choice(c, k, replace=repeat or k > c) for _ in range(n)]).astype(np.int32)
    t = (3 * rng.standard_normal((n, k)) + 5).astype(np.float32)
    return idx, t


def _run_distill(torch, vm, mode, x, idx, t, temp, gy, off=0):
    n, c = x.shape
    flat = torch.full((off + n * c,), NAN, device="cuda")
    flat[off:] = to_dev(torch, x).flatten()
    px = flat.data_ptr() + 4 * off
    y = torch.full((n,), NAN, device="cuda")
    gx = torch.full((n, c), NAN, device="cuda")
    ht = None if temp == 1.0 else torch.tensor([temp], device="cuda")
    di, dt, dg = to_dev(torch, idx), to_dev(torch, t), to_dev(torch, gy)
    if mode == "step":
        vm.softmax_top_distill_step(0, y, gx, dg, px, di, dt, n, c, idx.shape[1], ht)
    else:
        ps = torch.full((n, 3), NAN, device="cuda")
        vm.softmax_top_distill(0, y, ps, px, di, dt, n, c, idx.shape[1], ht)
        vm.softmax_top_distill_backward_x(0, gx, dg, px, ps, di, dt, n, c, idx.shape[1], ht)
    torch.cuda.synchronize()
    return to_host(y), to_host(gx)


def _near(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


SHAPES = [(1, 1, 1), (1, 2, 5), (3, 5, 5), (7, 33, 4), (2, 1000, 64), (5, 2047, 3), (3, 4099, 600), (1, 32000, 32),
          (2, 50257, 64), (300, 130, 8), (2, 128256, 17), (1, 131073, 9), (2, 140001, 40), (600, 2100, 1), (2, 300, 2048), (2, 380001, 1500),
          (1, 450001, 30), (700, 1030, 5)]


@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("shape", SHAPES)
def test_distill(torch_cuda, vm, shape, mode):
    n, c, k = shape
    rng = np.random.default_rng(n * 1000 + c + k)
    x = (2.5 * rng.standard_normal((n, c))).astype(np.float32)
    idx, t = _table(rng, n, c, k)
    temp = 2.0 if c % 2 else 1.0
    gy = rng.standard_normal(n).astype(np.float32)
    y, gx, ty, tg = _distill_truth(x, idx, t, temp, gy)
    got = _run_distill(torch_cuda, vm, mode, x, idx, t, temp, gy)
    _near(got[0], y, ty)
    _near(got[1], gx, tg)


@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_distill_alignments_repeats_and_gaps(torch_cuda, vm, off, mode):
    """Input rows off the 16-byte grid (and then out of step with the output's), ids that occur twice, unused entries."""
    rng = np.random.default_rng(off)
    n, c, k = 6, 4005, 40
    x = (2 * rng.standard_normal((n, c))).astype(np.float32)
    idx, t = _table(rng, n, c, k)
    idx[0, :k // 2] = idx[0, k // 2:]              # every id twice
    idx[1, 5:] = idx[1, 4]                         # one id 36 times
    idx[2, 1::2] = -1                              # gaps
    idx[3, :] = -1                                 # no entry at all
    t[4, 3:] = -np.inf                             # entries without weight
    t[5, :], x[5, :] = -np.inf, np.nan             # nothing has weight; the row's logits are not looked at
    t[2, 1::2] = np.nan                            # what stands in unused entries is not looked at
    x[3, :] = np.nan
    idx[0, 0] = c - 1
    idx[0, 1] = 0
    gy = rng.standard_normal(n).astype(np.float32)
    good = [0, 1, 2, 4]
    got = _run_distill(torch_cuda, vm, mode, x, idx, t, 1.5, gy, off)
    y, gx, ty, tg = _distill_truth(x[good], idx[good], t[good], 1.5, gy[good])
    _near(got[0][good], y, ty)
    _near(got[1][good], gx, tg)
    for r in (3, 5):
        assert got[0][r] == 0.0 and np.all(got[1][r] == 0.0)


@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("ncol", [40, 9000, 440001])
def test_distill_infinities(torch_cuda, vm, mode, ncol):
    """Logits of -inf (a masked vocabulary) have no probability; the type's lowest value behaves as such; a labelled -inf is an infinite
    loss; NaN and +inf poison their own row only."""
    rng = np.random.default_rng(ncol)
    x = rng.standard_normal((6, ncol)).astype(np.float32)
    idx, t = _table(rng, 6, ncol, 4)
    idx[:] = [[3, 7, 11, 2]]
    x[0, 12:] = -np.inf
    x[1, 12:] = np.finfo(np.float32).min
    x[2, 7] = -np.inf
    x[3, ncol - 1] = np.nan
    x[4, 20] = np.inf
    gy = np.ones(6, np.float32)
    y, gx = _run_distill(torch_cuda, vm, mode, x, idx, t, 1.0, gy)
    want = _distill_truth(x[[0, 1, 5]], idx[[0, 1, 5]], t[[0, 1, 5]], 1.0, gy)
    _near(y[[0, 1, 5]], want[0], want[2])
    _near(gx[[0, 1, 5]], want[1], want[3])
    assert np.all(gx[:2, 12:] == 0.0)
    assert y[2] == np.inf and np.all(np.isfinite(gx[2]))
    assert np.isnan(y[3]) and np.isnan(gx[3]).all()
    assert np.isnan(y[4])


@pytest.mark.parametrize("mode", ["step", "calls"])
def test_rows_without_a_distribution_and_tables_without_entries(torch_cuda, vm, mode):
    torch = torch_cuda
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 50)).astype(np.float32)
    x[0], x[1] = -np.inf, np.finfo(np.float32).min
    idx, t = _table(rng, 3, 50, 4)
    y, gx = _run_distill(torch, vm, mode, x, idx, t, 1.0, np.ones(3, np.float32))
    assert np.isnan(y[:2]).all() and np.isnan(gx[:2]).all() and np.isfinite(y[2]) and np.isfinite(gx[2]).all()
    y, gx = _run_distill(torch, vm, mode, x, np.zeros((3, 0), np.int32), np.zeros((3, 0), np.float32), 1.0, np.ones(3, np.float32))
    assert np.all(y == 0) and np.all(gx == 0)


def test_distill_gradient_against_differences(torch_cuda, vm):
    """Central differences of the kernel's own loss.  The loss is about 20, off by 1e-5 at most; h = 0.05 leaves h^2 / 6 times a third
    derivative below temp^-1 = 1/2 in size: 1e-5 / 0.05 + 0.0025 / 12 < 6e-4."""
    rng = np.random.default_rng(3)
    c, k, temp, h = 60, 6, 2.0, 0.05
    x0 = (2 * rng.standard_normal(c)).astype(np.float32)
    idx, t = _table(rng, 1, c, k)
    cols = np.concatenate([idx[0], np.setdiff1d(np.arange(c), idx[0])[:6]])
    x = np.repeat(x0[None], 2 * len(cols) + 1, 0)
    for i, col in enumerate(cols):
        x[2 * i, col] += np.float32(h)
        x[2 * i + 1, col] -= np.float32(h)
    n = len(x)
    y, gx = _run_distill(torch_cuda, vm, "step", x, np.repeat(idx, n, 0), np.repeat(t, n, 0), temp, np.ones(n, np.float32))
    for i, col in enumerate(cols):
        width = float(x[2 * i, col]) - float(x[2 * i + 1, col])
        assert abs((float(y[2 * i]) - float(y[2 * i + 1])) / width - gx[-1, col]) < 6e-4


# ---- policy loss -----------------------------------------------------------------------------------------
def _policy_truth(x, z, old, ref, adv, temp, gy, low, high, beta):
    n, c = x.shape
    q, logq, arg, rel = _soft(x, temp)
    l = logq[np.arange(n), z]
    el = rel[:, 0] + 3 * U * np.abs(arg[np.arange(n), z])      # error of l
    rho = np.exp(l - old) if old is not None else np.ones(n)
    er = rho * ((el if old is not None else 0) + 3 * U * (1 + (np.abs(l - old) if old is not None else 0)))
    bound = np.minimum(np.maximum(rho, 1 - low), 1 + high)
    free = rho * adv <= bound * adv
    y = -np.where(free, rho * adv, bound * adv)
    ty = np.abs(adv) * er + 4 * U * np.abs(y)
    slope = np.where(free, -adv * rho, 0.0)
    ts = np.abs(adv) * er * free + 4 * U * np.abs(slope)
    if ref is not None:
        d = ref - l
        em = np.expm1(d)
        y = y + beta * (em - d)
        slope = slope - beta * em
        ed = el + 2 * U * np.abs(d)
        ty = ty + beta * (np.abs(em) * ed + 4 * U * (np.abs(em) + np.abs(d)))
        ts = ts + beta * (np.exp(d) * ed + 4 * U * np.abs(em))
    hot = np.zeros((n, c))
    hot[np.arange(n), z] = 1
    k = gy * slope / temp
    gx = k[:, None] * (hot - q)
    tg = (np.abs(gy) * ts / temp)[:, None] * (hot + q) + np.abs(k)[:, None] * (
        q * ((3 * np.abs(arg) + 8) * U + rel) + 4 * U * hot) + 1e-38
    return y, l, gx, ty + 1e-38, el + 2 * U * np.abs(l), tg


def _run_policy(torch, vm, mode, x, z, old, ref, adv, temp, gy, low=0.2, high=0.3, beta=0.1):
    n, c = x.shape
    dev = lambda a: None if a is None else to_dev(torch, a)                                         # noqa: E731
    hyper = lambda v: None if v is None else torch.tensor([v], device="cuda")                       # noqa: E731
    y, logp = torch.full((n,), NAN, device="cuda"), torch.full((n,), NAN, device="cuda")
    gx = torch.full((n, c), NAN, device="cuda")
    hypers = [hyper(low), hyper(high), hyper(beta), hyper(temp)]
    dx, dz = dev(x), dev(z)
    if mode == "step":
        vm.softmax_policy_loss_step(0, y, logp, gx, dev(gy), dx, dz, dev(old), dev(ref), dev(adv), n, c, *hypers)
    else:
        ps = torch.full((n, 3), NAN, device="cuda")
        vm.softmax_policy_loss(0, y, logp, ps, dx, dz, dev(old), dev(ref), dev(adv), n, c, *hypers)
        vm.softmax_policy_loss_backward_x(0, gx, dev(gy), dx, ps, dz, n, c, hypers[3])
    torch.cuda.synchronize()
    return to_host(y), to_host(logp), to_host(gx)


def _policy_inputs(n, c, temp, seed):
    rng = np.random.default_rng(seed)
    x = (2 * rng.standard_normal((n, c))).astype(np.float32)
    z = rng.integers(0, c, n).astype(np.int32)
    now = _soft(x, temp)[1][np.arange(n), z]
    # ratios on all sides of the bounds, none closer to 0.8, 1.3 than the error of a ratio
    old = (now - np.log(rng.choice([0.5, 0.79, 0.81, 1.0, 1.2, 1.29, 1.31, 2.0], n))).astype(np.float32)
    ref = (now + 0.4 * rng.standard_normal(n)).astype(np.float32)
    adv = rng.standard_normal(n).astype(np.float32)
    gy = rng.standard_normal(n).astype(np.float32)
    return x, z, old, ref, adv, gy


@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("shape", [(1, 1), (9, 2), (40, 37), (3, 4097), (5, 32000), (2, 50257), (2, 128256), (1, 200003), (1, 460003),
                                   (700, 500)])
def test_policy(torch_cuda, vm, shape, mode):
    n, c = shape
    temp = 0.7 if c % 2 else 1.0
    x, z, old, ref, adv, gy = _policy_inputs(n, c, temp, n + c)
    for o, r in ((old, ref), (old, None), (None, ref)):
        want = _policy_truth(x, z, o, r, adv, temp, gy, 0.2, 0.3, 0.1)
        got = _run_policy(torch_cuda, vm, mode, x, z, o, r, adv, temp, gy)
        for a, w, tol in zip(got, want[:3], want[3:]):
            _near(a, w, tol)


@pytest.mark.parametrize("mode", ["step", "calls"])
def test_policy_rows_and_bounds(torch_cuda, vm, mode):
    n, c = 8, 300
    x, z, old, ref, adv, gy = _policy_inputs(n, c, 1.0, 5)
    z[1], x[1] = -1, np.nan                     # padding: nothing of the row is looked at
    z[2], old[2], ref[2], adv[2] = -1, np.nan, np.nan, np.nan
    adv[3], old[3] = 0.0, -2000.0               # no advantage, a ratio that overflows
    adv[4], old[4] = 1.5, -2000.0               # bounded from above
    got = _run_policy(torch_cuda, vm, mode, x, z, old, ref, adv, 1.0, gy)
    want = _policy_truth(np.nan_to_num(x), np.maximum(z, 0), np.maximum(np.nan_to_num(old), -700), np.nan_to_num(ref),
                         np.nan_to_num(adv), 1.0, gy, 0.2, 0.3, 0.1)
    for r in (1, 2):
        assert got[0][r] == 0 and got[1][r] == 0 and np.all(got[2][r] == 0)
    live = [0, 3, 4, 5, 6, 7]
    for a, w, tol in zip(got, want[:3], want[3:]):
        _near(a[live], w[live], tol[live] if tol[live].ndim == 1 else np.where(np.isfinite(tol[live]), tol[live], 1e-6))
    # no bounds, no KL coefficient
    z, x, old = np.maximum(z, 0), np.nan_to_num(x), np.zeros(n, np.float32) - 5
    got = _run_policy(torch_cuda, vm, mode, x, z, old, np.zeros(n, np.float32), np.ones(n, np.float32), 1.0, gy, None, None, None)
    want = _policy_truth(x, z, old, None, np.ones(n, np.float32), 1.0, gy, np.inf, np.inf, 0.0)
    for a, w, tol in zip(got, want[:3], want[3:]):
        _near(a, w, tol)


def test_policy_without_a_coefficient_ignores_the_reference(torch_cuda, vm):
    n, c = 4, 64
    x, z, old, ref, adv, gy = _policy_inputs(n, c, 1.0, 8)
    ref[1] = 1e5                                  # e^d overflows
    for mode in ("step", "calls"):
        got = _run_policy(torch_cuda, vm, mode, x, z, old, ref, adv, 1.0, gy, beta=0.0)
        want = _policy_truth(x, z, old, None, adv, 1.0, gy, 0.2, 0.3, 0.0)
        for a, w, tol in zip(got, want[:3], want[3:]):
            _near(a, w, tol)


def test_more_logits_than_32_bits_count(torch_cuda, vm):
    """2.2e9 logits, gradient in place: the last rows land where they belong."""
    torch = torch_cuda
    n, c = 66000, 32771
    x = torch.zeros((n, c), device="cuda")
    z = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    adv, y = torch.ones(n, device="cuda"), torch.empty(n, device="cuda")
    rows = [0, 32768, n - 2, n - 1]
    z[rows] = torch.tensor([5, 6, c - 1, 0], dtype=torch.int32, device="cuda")
    x[rows, :3] = torch.tensor([1.0, -2.0, 3.0], device="cuda")
    head = x[rows].cpu().numpy()
    vm.softmax_policy_loss_step(0, y, None, x, None, x, z, None, None, adv, n, c)
    torch.cuda.synchronize()
    want = _policy_truth(head, z[rows].cpu().numpy(), None, None, np.ones(4, np.float32), 1.0, np.ones(4, np.float32), np.inf, np.inf, 0.0)
    _near(to_host(x[rows]), want[2], want[5])
    assert float(x[1:1000].abs().max()) == 0.0 and float(x[n - 1000: n - 2].abs().max()) == 0.0


def test_policy_gradient_against_differences(torch_cuda, vm):
    """The loss is of size 1, off by 2e-6; h = 0.02, third derivative below 2: 2e-6 / 0.02 + 0.0004 / 3 < 3e-4."""
    c, h = 30, 0.02
    x, z, old, ref, adv, gy = _policy_inputs(1, c, 1.0, 11)
    adv[:] = -1.0
    cols = [int(z[0])] + [i for i in range(6) if i != z[0]]
    rows = np.repeat(x, 2 * len(cols) + 1, 0)
    for i, col in enumerate(cols):
        rows[2 * i, col] += np.float32(h)
        rows[2 * i + 1, col] -= np.float32(h)
    n = len(rows)
    rep = lambda a: np.repeat(a, n)                                                                 # noqa: E731
    y, _, gx = _run_policy(torch_cuda, vm, "calls", rows, rep(z), rep(old), rep(ref), rep(adv), 1.0, np.ones(n, np.float32),
                           None, None, 0.1)
    for i, col in enumerate(cols):
        width = float(rows[2 * i, col]) - float(rows[2 * i + 1, col])
        assert abs((float(y[2 * i]) - float(y[2 * i + 1])) / width - gx[-1, col]) < 3e-4


# ---- both ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("ncol", [7, 50257, 440001])
def test_gradient_over_the_logits_and_default_gradient(torch_cuda, vm, ncol):
    """pgx = px, and pgy = NULL: the same bits as with buffers of their own and a gradient of ones."""
    torch = torch_cuda
    n, k = 5, 7
    rng = np.random.default_rng(ncol)
    x = to_dev(torch, (2 * rng.standard_normal((n, ncol))).astype(np.float32))
    idx, t = (to_dev(torch, a) for a in _table(rng, n, ncol, k))
    z, adv = idx[:, 0].contiguous(), torch.ones(n, device="cuda")
    one, y, ps = torch.ones(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty((n, 3), device="cuda")

    calls = [
        lambda px, gx, gy: vm.softmax_top_distill_step(0, y, gx, gy, px, idx, t, n, ncol, k),
        lambda px, gx, gy: (vm.softmax_top_distill(0, y, ps, px, idx, t, n, ncol, k),
                            vm.softmax_top_distill_backward_x(0, gx, gy, px, ps, idx, t, n, ncol, k)),
        lambda px, gx, gy: vm.softmax_policy_loss_step(0, y, None, gx, gy, px, z, None, None, adv, n, ncol),
        lambda px, gx, gy: (vm.softmax_policy_loss(0, y, None, ps, px, z, None, None, adv, n, ncol),
                            vm.softmax_policy_loss_backward_x(0, gx, gy, px, ps, z, n, ncol)),
    ]
    for call in calls:
        want = torch.full_like(x, NAN)
        call(x, want, one)
        over = x.clone()
        call(over, over, None)
        torch.cuda.synchronize()
        assert torch.equal(want, over)


def test_labels_out_of_range(torch_cuda, pkg, vm):
    """The row turns NaN, its neighbours keep their values, and the status call reports it once."""
    torch = torch_cuda
    rng = np.random.default_rng(0)
    n, c = 4, 100
    x = rng.standard_normal((n, c)).astype(np.float32)
    idx, t = _table(rng, n, c, 3)
    gy = np.ones(n, np.float32)
    lib = pkg.load()
    assert lib.kai_device_status(0, None) == 0
    for bad in (c, -2, 2 ** 31 - 1):
        for mode in ("step", "calls"):
            idx2 = idx.copy()
            idx2[2, 1] = bad
            y, gx = _run_distill(torch, vm, mode, x, idx2, t, 1.0, gy)
            assert lib.kai_device_status(0, None) == pkg.capi.E_OUT_OF_RANGE
            assert lib.kai_device_status(0, None) == 0
            assert np.isnan(y[2]) and np.isnan(gx[2]).all()
            assert np.isfinite(y[[0, 1, 3]]).all() and np.isfinite(gx[[0, 1, 3]]).all()
            z = np.array([1, bad, 2, 3], np.int32)
            y, logp, gx = _run_policy(torch, vm, mode, x, z, None, None, gy, 1.0, gy)
            assert lib.kai_device_status(0, None) == pkg.capi.E_OUT_OF_RANGE
            assert np.isnan(y[1]) and np.isnan(logp[1]) and np.isnan(gx[1]).all() and np.isfinite(gx[[0, 2, 3]]).all()
    assert lib.kai_device_status_clear(0) == 0


def test_rows_behind_the_last_keep_their_values(torch_cuda, vm):
    torch = torch_cuda
    n, c, k = 3, 1001, 4
    rng = np.random.default_rng(2)
    x = to_dev(torch, rng.standard_normal((n, c)).astype(np.float32))
    idx, t = (to_dev(torch, a) for a in _table(rng, n, c, k))
    gx, y = torch.full((n + 1, c), 5.0, device="cuda"), torch.full((n + 1,), 5.0, device="cuda")
    vm.softmax_top_distill_step(0, y, gx, None, x, idx, t, n, c, k)
    vm.softmax_top_distill_step(0, y, gx, None, x, idx, t, 0, c, k)
    torch.cuda.synchronize()
    assert float(y[n]) == 5.0 and bool((gx[n] == 5.0).all())


# Sizes on both sides of what a warp's registers hold, label counts on both sides of what one warp joins.
@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("shape", [(37, 256, 9), (21, 257, 64), (19, 512, 130), (23, 513, 33), (17, 1024, 256), (15, 1025, 257), (13, 2048, 128),
                                   (11, 2049, 129), (9, 2047, 700), (2500, 70, 300), (640, 2500, 40), (13, 4096, 70), (11, 4097, 256)])
def test_distill_repeats_at_every_size(torch_cuda, vm, shape, mode):
    """Rows with repeated ids, with distinct ones and with gaps next to one another, whatever kernel takes them."""
    n, c, k = shape
    rng = np.random.default_rng(n + c + k)
    x = (2.5 * rng.standard_normal((n, c))).astype(np.float32)
    idx, t = _table(rng, n, c, k, repeat=True)
    for r in range(0, n, 3):
        m = min(k, c)
        idx[r, :m], idx[r, m:] = rng.permutation(c)[:m], -1
    idx[1::3][rng.random(idx[1::3].shape) < 0.3] = -1
    temp = 2.0 if c % 2 else 1.0
    gy = rng.standard_normal(n).astype(np.float32)
    y, gx, ty, tg = _distill_truth(x, idx, t, temp, gy)
    for off in (0, 1):
        got = _run_distill(torch_cuda, vm, mode, x, idx, t, temp, gy, off)
        _near(got[0], y, ty)
        _near(got[1], gx, tg)


@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("ncol", [2048, 128256])
def test_distill_ids_that_a_hash_puts_together(torch_cuda, vm, mode, ncol):
    """Distinct ids with the same leading bits of a multiplicative hash, alone and with one of them repeated."""
    z = np.arange(ncol, dtype=np.uint64)
    near = z[(z * 2654435761 % 2 ** 32) < 2 ** 32 * 24 // ncol].astype(np.int32)
    n, k = 4, len(near) + 1
    assert k >= 16
    rng = np.random.default_rng(ncol)
    x = (2 * rng.standard_normal((n, ncol))).astype(np.float32)
    _, t = _table(rng, n, ncol, k)
    idx = np.stack([np.append(near, -1), np.append(near, near[0]), np.append(near, near[-1])[::-1], np.append(near[::-1], near[3])]).astype(np.int32)
    gy = rng.standard_normal(n).astype(np.float32)
    y, gx, ty, tg = _distill_truth(x, idx, t, 1.0, gy)
    got = _run_distill(torch_cuda, vm, mode, x, idx, t, 1.0, gy)
    _near(got[0], y, ty)
    _near(got[1], gx, tg)


def test_distill_more_rows_than_warps(torch_cuda, vm):
    n, c, k = 41003, 5, 3
    rng = np.random.default_rng(n)
    x = (2 * rng.standard_normal((n, c))).astype(np.float32)
    idx, t = rng.integers(-1, c, (n, k)).astype(np.int32), rng.standard_normal((n, k)).astype(np.float32)
    gy = rng.standard_normal(n).astype(np.float32)
    y, gx, ty, tg = _distill_truth(x, idx, t, 1.0, gy)
    got = _run_distill(torch_cuda, vm, "step", x, idx, t, 1.0, gy)
    _near(got[0], y, ty)
    _near(got[1], gx, tg)


@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("shape", [(41003, 9), (70, 256), (61, 257), (51, 512), (41, 513), (33, 1024), (31, 1025), (27, 2048), (25, 2049), (14, 4096)])
def test_policy_at_every_size(torch_cuda, vm, shape, mode):
    n, c = shape
    x, z, old, ref, adv, gy = _policy_inputs(n, c, 1.0, n * c)
    want = _policy_truth(x, z, old, ref, adv, 1.0, gy, 0.2, 0.3, 0.1)
    z = z.copy()
    gone = np.arange(n) % 7 == 6
    z[gone] = -1                                   # padding
    got = _run_policy(torch_cuda, vm, mode, x, z, old, ref, adv, 1.0, gy)
    for a, w, tol in zip(got, want[:3], want[3:]):
        _near(a[~gone], w[~gone], tol[~gone])
        assert np.all(a[gone] == 0.0)


@pytest.mark.parametrize("ncol", [300, 1500])
def test_short_rows_with_bad_labels_keep_their_neighbours(torch_cuda, pkg, vm, ncol):
    """One bad id among many labels and rows: that row is NaN, all others are as without it."""
    torch = torch_cuda
    rng = np.random.default_rng(ncol)
    n, k = 45, 200
    x = rng.standard_normal((n, ncol)).astype(np.float32)
    idx, t = _table(rng, n, ncol, k)
    gy = np.ones(n, np.float32)
    lib = pkg.load()
    for mode in ("step", "calls"):
        assert lib.kai_device_status_clear(0) == 0
        want = _run_distill(torch, vm, mode, x, idx, t, 1.0, gy)
        worse = idx.copy()
        worse[20, 150], worse[21, 3] = ncol, -7
        got = _run_distill(torch, vm, mode, x, worse, t, 1.0, gy)
        assert lib.kai_device_status(0, None) == pkg.capi.E_OUT_OF_RANGE
        rest = np.delete(np.arange(n), [20, 21])
        assert all(np.array_equal(a[rest], b[rest]) and np.isnan(a[20:22]).all() for a, b in zip(got, want))
    assert lib.kai_device_status_clear(0) == 0
