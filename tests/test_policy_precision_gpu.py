"""The digits of the policy loss where they can be told apart from those of the row's sum.

Every logit is 0 and the number of columns a power of two, 2^n: all exponentials are 1 and their sum is exact, so that a token's
log-probability is -n ln 2 to 64 bits (off by 2^-52 |l| < 3e-15), and q = 2^-n exactly.  What is left is the loss's own arithmetic."""
import numpy as np
import pytest

from helpers import to_dev, to_host

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24 * (1 + 2.0 ** -20)      # one fp32 rounding, relative


def _run(torch, vm, mode, n, ncol, z, old, ref, adv, beta):
    dev = lambda a: None if a is None else to_dev(torch, a)                                         # noqa: E731
    x, dz = torch.zeros((n, ncol), device="cuda"), dev(z)
    y, gx = torch.full((n,), float("nan"), device="cuda"), torch.full((n, ncol), float("nan"), device="cuda")
    hyper = None if beta is None else torch.tensor([beta], device="cuda")
    d_old, d_ref, d_adv = dev(old), dev(ref), dev(adv)
    if mode == "step":
        vm.softmax_policy_loss_step(0, y, None, gx, None, x, dz, d_old, d_ref, d_adv, n, ncol, None, None, hyper)
    else:
        ps = torch.empty((n, 3), device="cuda")
        vm.softmax_policy_loss(0, y, None, ps, x, dz, d_old, d_ref, d_adv, n, ncol, None, None, hyper)
        vm.softmax_policy_loss_backward_x(0, gx, None, x, ps, dz, n, ncol)
    torch.cuda.synchronize()
    rows = torch.arange(n, device="cuda")
    other = gx[rows, (dz.long() + 1) % ncol]
    return to_host(y).astype(np.float64), to_host(gx[rows, dz.long()]).astype(np.float64), to_host(other).astype(np.float64)


# a warp's row, a CTA's, a cluster's, and a row that no cluster holds
SIZES = [64, 8192, 131072, 524288]


@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("ncol", SIZES)
def test_kl_term_next_to_the_reference(torch_cuda, vm, ncol, mode):
    """Without an advantage the loss is e^d - d - 1, about d^2 / 2.  Its 64-bit form is off by 2^-52 |d| and by the error of l times
    |d|, below 1e-10 of it from |d| = 1e-4 on; what remains is the rounding of the term and of the sum it joins: two.  The gradient's
    e^d - 1: d rounded, expm1f within a unit in the last place, three more roundings on the way to the column."""
    l = -np.log2(ncol) * np.log(2.0)
    target = np.array([s * d for d in (0.7, 0.1, 1e-2, 3e-3, 1e-3, 3e-4, 1e-4) for s in (1, -1)])
    n = len(target)
    ref = (l + target).astype(np.float32)
    d = ref.astype(np.float64) - l
    z = (np.arange(n) * 7 % ncol).astype(np.int32)
    y, at, other = _run(torch_cuda, vm, mode, n, ncol, z, None, ref, np.zeros(n, np.float32), 1.0)
    dl = d.astype(np.longdouble)
    want = (np.expm1(dl) - dl).astype(np.float64)
    assert np.all(np.abs(y - want) <= 2 * HALF * want), np.abs(y / want - 1).max()
    slope = -np.expm1(d)
    assert np.all(np.abs(other + slope / ncol) <= 7 * HALF * np.abs(slope) / ncol)
    assert np.all(np.abs(at - slope * (1 - 1 / ncol)) <= 8 * HALF * np.abs(slope))


@pytest.mark.parametrize("mode", ["step", "calls"])
@pytest.mark.parametrize("ncol", SIZES)
def test_ratio(torch_cuda, vm, ncol, mode):
    """Advantage -1, no bounds, ratios from e^-12 to e^12: the loss is the ratio e^(l - old) itself: expf of the rounded difference (a unit in the last place: 2 u)
    times 1 plus what the rounding lost (two roundings; the square of 2^-23 left out).  The gradient's columns are it times q
    (exact) beside the label's, and its difference to that, rounded again, at the label."""
    n = 16 if ncol > 8192 else 1500
    l = -np.log2(ncol) * np.log(2.0)
    old = (l + np.random.default_rng(ncol).uniform(-12, 12, n)).astype(np.float32)
    rho = np.exp(l - old.astype(np.float64))
    z = (np.arange(n) * 7 % ncol).astype(np.int32)
    y, at, other = _run(torch_cuda, vm, mode, n, ncol, z, old, None, -np.ones(n, np.float32), None)
    assert np.all(np.abs(y - rho) <= 4 * HALF * rho), np.abs(y / rho - 1).max()
    assert np.all(np.abs(other + rho / ncol) <= 4 * HALF * rho / ncol)
    assert np.all(np.abs(at - rho * (1 - 1 / ncol)) <= 5 * HALF * rho)
