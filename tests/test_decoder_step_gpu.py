"""The decoder-training operators together, as a training step uses them: rotary positions in front of the framework's attention,
the gated layer with its down projection, logits, and one of the losses on them; forward and backward, against
torch's gradients in 64 bits; recorded as one call list; on a stream of its own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NBAT, T, NHEAD, P, F, V, K, NROT = 2, 33, 4, 16, 96, 211, 8, 12
C, M = NHEAD * P, NBAT * T


def _weights(torch):
    gen = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(s, device="cuda", generator=gen)       # noqa: E731
    w = {"x": r(M, C), "wq": r(C, C) / 8, "wk": r(C, C) / 8, "wv": r(C, C) / 8, "wg": r(F, C) / 8, "wu": r(F, C) / 8, "wd": r(C, F) / 10,
         "wo": r(V, C) / 8}
    idx = torch.stack([torch.randperm(V, device="cuda", generator=gen)[:K] for _ in range(M)]).int()
    idx[::5] = -1                                                      # padded tokens
    idx[1::3, K // 2:] = -1
    t = 2 * r(M, K)
    gy = r(M)
    z = torch.where(idx[:, 0] >= 0, idx[:, 1], -1).int().contiguous()
    return w, idx, t, gy, z, r(M) - 5, r(M) - 5, r(M)


class Step:
    """Buffers of one step, and the calls that fill them."""

    def __init__(self, torch, vm, loss):
        self.torch, self.vm, self.loss = torch, vm, loss
        self.w, self.idx, self.t, self.gy, self.z, self.old, self.ref, self.adv = _weights(torch)
        e = lambda *s: torch.full(s, float("nan"), device="cuda")     # noqa: E731
        self.freq = torch.empty(NROT // 2, device="cuda", dtype=torch.float64)
        vm.rotary_frequencies(0, self.freq, NROT, 1000.0, "by_parts", 4.0, 1.0, 32.0, 64)
        self.q, self.k, self.v, self.at = e(M, C), e(M, C), e(M, C), e(M, C)
        self.probs, self.gp = e(NBAT, T, T, NHEAD), e(NBAT, T, T, NHEAD)
        self.h, self.g, self.u, self.gg, self.gu, self.gh = (e(M, F) for _ in range(6))
        self.o, self.go, self.ga, self.gq, self.gk, self.gv = (e(M, C) for _ in range(6))
        self.logits, self.gl, self.y = e(M, V), e(M, V), e(M)
        self.grads = {n: torch.full_like(v, float("nan")) for n, v in self.w.items()}
        self.coef = torch.tensor([P ** -0.5], device="cuda")
        self.hyper = [torch.tensor([v], device="cuda") for v in (0.2, 0.3, 0.05, 1.5)]

    def run(self, s=None):
        vm, w, g = self.vm, self.w, self.grads
        for out, name in ((self.q, "wq"), (self.k, "wk"), (self.v, "wv")):
            vm.matmul(0, out, w[name], w["x"], C, M, C, stream=s)
        for r in (self.q, self.k):
            vm.rotary(0, r, r, self.freq, None, 100, NBAT, T, NHEAD, P, NROT, "half", stream=s)
        dims = (NBAT, T, C, NHEAD, P)
        vm.mult_on_heads(0, self.probs, self.k, self.q, *dims, self.coef, stream=s)
        vm.set_mh_attention_mask(0, self.probs, NBAT, T, NHEAD, True, stream=s)
        vm.softmax_direct_on_axis(0, self.probs, M, T, NHEAD, stream=s)
        vm.mix_values(0, self.at, self.probs, self.v, *dims, stream=s)
        vm.gated_linear_forward(0, self.h, self.g, self.u, w["wg"], w["wu"], self.at, None, None, F, M, C, "swish", stream=s)
        vm.matmul(0, self.o, w["wd"], self.h, C, M, F, stream=s)
        vm.matmul(0, self.logits, w["wo"], self.o, V, M, C, stream=s)
        if self.loss == "distill":
            vm.softmax_top_distill_step(0, self.y, self.gl, self.gy, self.logits, self.idx, self.t, M, V, K, self.hyper[3], stream=s)
        else:
            vm.softmax_policy_loss_step(0, self.y, None, self.gl, self.gy, self.logits, self.z, self.old, self.ref, self.adv, M, V,
                                        *self.hyper, stream=s)
        vm.matmul_backward_w(0, g["wo"], self.gl, self.o, V, M, C, stream=s)
        vm.matmul_backward_x(0, self.go, self.gl, w["wo"], V, M, C, stream=s)
        vm.matmul_backward_w(0, g["wd"], self.go, self.h, C, M, F, stream=s)
        vm.matmul_backward_x(0, self.gh, self.go, w["wd"], C, M, F, stream=s)
        vm.gated_linear_backward(0, self.ga, g["wg"], g["wu"], self.gg, self.gu, self.gh, self.g, self.u, w["wg"], w["wu"], self.at,
                                 F, M, C, "swish", stream=s)
        vm.mix_values_backward_value(0, self.gv, self.ga, self.probs, *dims, stream=s)
        vm.mix_values_backward_prop(0, self.gp, self.ga, self.v, *dims, stream=s)
        vm.softmax_direct_on_axis_backward(0, self.gp, self.probs, NBAT, T, NHEAD, self.coef, stream=s)
        vm.mult_on_heads_backward(0, self.gq, self.gp, self.k, *dims, stream=s)
        # the key's gradient is the transposed contraction
        vm.mix_values_backward_value(0, self.gk, self.q, self.gp, *dims, stream=s)
        for r in (self.gq, self.gk):
            vm.rotary_backward(0, r, r, self.freq, None, 100, NBAT, T, NHEAD, P, NROT, "half", stream=s)
        for i, (gr, name) in enumerate(((self.gq, "wq"), (self.gk, "wk"), (self.gv, "wv"))):
            vm.matmul_backward_w(0, g[name], gr, w["x"], C, M, C, stream=s)
            vm.matmul_backward_x(0, g["x"], gr, w[name], C, M, C, acc=i > 0, stream=s)

    def truth(self):
        torch = self.torch
        w = {n: v.double().requires_grad_() for n, v in self.w.items()}

        def turn(x):
            x = x.view(NBAT, T, NHEAD, P)
            ang = (100 + torch.arange(T, device="cuda")).double()[None, :, None, None] * self.freq
            a, b, rest = x[..., : NROT // 2], x[..., NROT // 2: NROT], x[..., NROT:]
            return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), rest], -1)

        q, k = turn(w["x"] @ w["wq"].T), turn(w["x"] @ w["wk"].T)
        v = (w["x"] @ w["wv"].T).view(NBAT, T, NHEAD, P)
        score = torch.einsum("bqhp,bkhp->bhqk", q, k) * P ** -0.5
        score = score.masked_fill(torch.ones(T, T, device="cuda").triu(1).bool(), -np.inf)
        at = torch.einsum("bhqk,bkhp->bqhp", score.softmax(-1), v).reshape(M, C)
        h = torch.nn.functional.silu(at @ w["wg"].T) * (at @ w["wu"].T)
        logits = (h @ w["wd"].T) @ w["wo"].T
        logq = (logits / 1.5).log_softmax(-1)
        if self.loss == "distill":
            live = (self.idx >= 0).any(-1)
            t = torch.where((self.idx >= 0) | ~live[:, None], self.t.double() / 1.5, -np.inf)
            logp = t.log_softmax(-1)
            p = logp.exp()
            y = 1.5 ** 2 * (p * (torch.where(p > 0, logp, 0.0) - logq.gather(1, self.idx.long().clamp(min=0)))).sum(-1)
        else:
            live = self.z >= 0
            l = logq.gather(1, self.z.long().clamp(min=0)[:, None])[:, 0]
            rho, adv, d = (l - self.old.double()).exp(), self.adv.double(), self.ref.double() - l
            low, high, beta = (float(x) for x in self.hyper[:3])
            y = -torch.minimum(rho * adv, rho.clamp(1 - low, 1 + high) * adv) + beta * (torch.expm1(d) - d)
        y = torch.where(live, y, 0.0)
        return y.detach(), dict(zip(w, torch.autograd.grad(y, list(w.values()), self.gy.double())))


@pytest.mark.parametrize("loss", ["distill", "policy"])
def test_training_step(torch_cuda, vm, loss):
    """About ten operators in a row, each off by less than 2e-6 of its result (their own tests), gains of order one between them:
    2e-5 of each gradient's norm."""
    s = Step(torch_cuda, vm, loss)
    s.run()
    torch_cuda.cuda.synchronize()
    y, grads = s.truth()
    assert float((s.y.double() - y).norm() / y.norm()) <= 2e-5
    for n, want in grads.items():
        assert float((s.grads[n].double() - want).norm() / want.norm()) <= 2e-5, n


@pytest.mark.parametrize("loss", ["distill", "policy"])
def test_recorded_step(torch_cuda, pkg, vm, loss):
    """The step as one recorded list, replayed on new inputs, equals the calls one by one bit for bit -- before and after ordinary calls
    that need more scratch memory than the recorded ones."""
    torch = torch_cuda
    s = Step(torch, vm, loss)
    s.run()
    with vm.Replay(0) as rp:
        s.run(rp.stream)
    try:
        for seed in range(2):
            s.w["x"].copy_(torch.randn((M, C), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
            s.run()
            torch.cuda.synchronize()
            want = {n: v.clone() for n, v in s.grads.items()}
            want_y = s.y.clone()
            for v in s.grads.values():
                v.fill_(float("nan"))
            torch.cuda.synchronize()
            rp.launch()
            torch.cuda.synchronize()
            assert torch.equal(s.y, want_y)
            assert all(torch.equal(s.grads[n], want[n]) for n in want)
            big = torch.randn((1024, 512), device="cuda")
            w1, w2 = torch.randn((768, 512), device="cuda"), torch.randn((768, 512), device="cuda")
            out = torch.empty((1024, 768), device="cuda")
            vm.gated_linear_forward(0, out, None, None, w1, w2, big, None, None, 768, 1024, 512, "swish")
        assert pkg.load().kai_device_status(0, None) == 0
    finally:
        rp.close()


def test_stream_of_its_own(torch_cuda, vm):
    """Calls on a side stream are ordered with that stream's other work."""
    torch = torch_cuda
    s = Step(torch, vm, "distill")
    s.run()
    torch.cuda.synchronize()
    want = {n: v.clone() for n, v in s.grads.items()}
    x = s.w["x"].clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        s.w["x"].copy_(x)
        for v in s.grads.values():
            v.fill_(float("nan"))
        s.run(side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(s.grads[n], want[n]) for n in want)
