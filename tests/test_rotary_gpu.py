"""Rotary positions against the complex product in 64 bits.

Tolerance of one value, per unit of |a| + |b| (times the scale): the remainder in turns is rounded to fp32 (9.4e-8
radians), sincospif is off by an ulp (1.2e-7), the scale, the product and the fused sum round once each (3 x 6e-8):
4e-7, and 2 pi * 3 * 2^-53 per turn of the angle."""
import numpy as np
import pytest

from helpers import to_dev, to_host

pytestmark = pytest.mark.gpu

SHAPES = [  # nbat, ntimes, nhead, npiece, nrot
    (1, 1, 1, 2, 2), (1, 1, 8, 64, 64), (2, 5, 3, 64, 32), (3, 7, 2, 80, 40), (1, 33, 5, 10, 6), (2, 9, 4, 7, 4),
    (1, 3, 2, 16, 0), (2, 2, 1, 12, 12), (1, 2049, 8, 64, 64), (4, 100, 12, 20, 20), (1, 1, 1, 3, 2), (5, 1, 24, 128, 64),
]


def _truth(x, pos, freq, half, scale, sign=1.0):
    x = x.astype(np.float64)
    r = 2 * len(freq)
    t = pos.astype(np.float64)[..., None, None] * freq * sign
    a, b = (x[..., : r // 2], x[..., r // 2: r]) if half else (x[..., 0:r:2], x[..., 1:r:2])
    z = (a + 1j * b) * np.exp(1j * t) * scale
    out = x.copy()
    if half:
        out[..., : r // 2], out[..., r // 2: r] = z.real, z.imag
    else:
        out[..., 0:r:2], out[..., 1:r:2] = z.real, z.imag
    size = np.zeros_like(x)
    s = (np.abs(a) + np.abs(b)) * scale * (4e-7 + 2 * np.pi * 3 * 2.0 ** -53 * np.abs(t) / (2 * np.pi))
    if half:
        size[..., : r // 2] = size[..., r // 2: r] = s
    else:
        size[..., 0:r:2] = size[..., 1:r:2] = s
    return out, size


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradient(torch_cuda, vm, shape, layout):
    torch = torch_cuda
    nbat, ntimes, nhead, npiece, nrot = shape
    rng = np.random.default_rng(npiece * 7 + nrot)
    x = rng.standard_normal((nbat, ntimes, nhead, npiece)).astype(np.float32)
    freq = 10000.0 ** (-2.0 * np.arange(nrot // 2) / max(nrot, 1))
    pos = rng.integers(-50, 1_000_000, (nbat, ntimes))
    dx, df, dp = to_dev(torch, x), to_dev(torch, freq), to_dev(torch, pos)
    scale = torch.tensor([1.25], device="cuda")
    for call, sign, hs in ((vm.rotary, 1.0, None), (vm.rotary_backward, -1.0, scale)):
        y = torch.full_like(dx, float("nan"))
        call(0, y, dx, df, dp, 12345, nbat, ntimes, nhead, npiece, nrot, layout, hs)
        torch.cuda.synchronize()
        want, tol = _truth(x, pos, freq, layout == "half", 1.25 if hs is not None else 1.0, sign)
        assert np.all(np.abs(to_host(y) - want) <= tol)
        # positions as an offset
        y.fill_(float("nan"))
        call(0, y, dx, df, None, 77, nbat, ntimes, nhead, npiece, nrot, layout, hs)
        torch.cuda.synchronize()
        at = np.broadcast_to(77 + np.arange(ntimes), (nbat, ntimes))
        want, tol = _truth(x, at, freq, layout == "half", 1.25 if hs is not None else 1.0, sign)
        assert np.all(np.abs(to_host(y) - want) <= tol)
        # in place
        z = dx.clone()
        call(0, z, z, df, None, 77, nbat, ntimes, nhead, npiece, nrot, layout, hs)
        torch.cuda.synchronize()
        assert torch.equal(z, y)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_packed_projection(torch_cuda, vm, layout, offset):
    """q and k turned where they lie in rows of [q | k | v], in place, at every alignment; v and the gaps keep their bits."""
    torch = torch_cuda
    rows, nhead, npiece, nrot = 37, 6, 24, 16
    ld = 3 * nhead * npiece // 2 + 5 * offset        # 4 heads' worth of q and k together, then v
    nqk = 4
    rng = np.random.default_rng(offset)
    buf = rng.standard_normal(offset + rows * ld).astype(np.float32)
    d = to_dev(torch, buf)
    freq = 500.0 ** (-np.arange(nrot // 2) / (nrot // 2))
    at = d.data_ptr() + 4 * offset
    vm.rotary(0, at, at, to_dev(torch, freq), None, 3, 1, rows, nqk, npiece, nrot, layout, ldy=ld, ldx=ld)
    torch.cuda.synchronize()
    got = to_host(d)[offset:].reshape(rows, ld)
    src = buf[offset:].reshape(rows, ld)
    want, tol = _truth(src[:, : nqk * npiece].reshape(1, rows, nqk, npiece), 3 + np.arange(rows)[None], freq,
                       layout == "half", 1.0)
    assert np.all(np.abs(got[:, : nqk * npiece] - want.reshape(rows, -1)) <= tol.reshape(rows, -1))
    np.testing.assert_array_equal(got[:, nqk * npiece:], src[:, nqk * npiece:])
    np.testing.assert_array_equal(to_host(d)[:offset], buf[:offset])


def test_gradient_is_the_transpose(torch_cuda, vm):
    """<R x, g> = <x, R^T g> summed in 64 bits, for both layouts."""
    torch = torch_cuda
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, g = (torch.randn((2, 50, 4 * 48), device="cuda", generator=gen) for _ in range(2))
    freq = torch.tensor(10000.0 ** (-np.arange(16) / 16), device="cuda")
    for layout in ("half", "interleaved"):
        y, gx = torch.empty_like(x), torch.empty_like(x)
        vm.rotary(0, y, x, freq, None, 1000, 2, 50, 4, 48, 32, layout)
        vm.rotary_backward(0, gx, g, freq, None, 1000, 2, 50, 4, 48, 32, layout)
        torch.cuda.synchronize()
        left, right = (y.double() * g.double()).sum(), (x.double() * gx.double()).sum()
        size = (x.double().abs() * g.double().abs()).sum()
        assert abs(float(left - right)) <= 2 * 4e-7 * 2 * float(size)


@pytest.mark.parametrize("scaling", ["plain", "linear", "base", "by_parts"])
@pytest.mark.parametrize("nrot", [4, 64, 130])
def test_frequencies(torch_cuda, vm, scaling, nrot):
    torch = torch_cuda
    base, factor, slow, fast, times = 50000.0, 6.5, 1.0, 32.0, 4096
    out = torch.full((nrot // 2,), float("nan"), device="cuda", dtype=torch.float64)
    vm.rotary_frequencies(0, out, nrot, base, scaling, factor, slow, fast, times)
    torch.cuda.synchronize()
    e = np.arange(nrot // 2) * 2.0 / nrot
    f = (base * factor ** (nrot / (nrot - 2)) if scaling == "base" else base) ** -e
    if scaling == "linear":
        f = f / factor
    if scaling == "by_parts":
        keep = np.clip((times * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        f = f * (keep + (1 - keep) / factor)
    # pow is within two units in the last place on both sides, a few products round; `base` raises its error to e <= 1
    np.testing.assert_allclose(to_host(out), f, rtol=16 * 2.0 ** -52)


def test_long_offsets(torch_cuda, vm):
    """A tensor of more than 2^31 values: its last row is turned where it lies, rows in front of it too."""
    torch = torch_cuda
    nvec, rows = 4096, (1 << 19) + 3
    x = torch.zeros((rows, nvec), device="cuda")
    x[-1], x[1 << 18] = 1.0, 2.0
    freq = torch.tensor(10000.0 ** (-np.arange(32) / 32), device="cuda")
    vm.rotary(0, x, x, freq, None, 0, 1, rows, 64, 64, 64, "half")
    torch.cuda.synchronize()
    for row, v in ((rows - 1, 1.0), (1 << 18, 2.0)):
        want, tol = _truth(np.full((1, 1, 64, 64), v, np.float32), np.array([[row]]), to_host(freq), True, 1.0)
        assert np.all(np.abs(to_host(x[row]).reshape(want.shape) - want) <= tol)
    assert float(x[: 1 << 18].abs().max()) == 0.0
