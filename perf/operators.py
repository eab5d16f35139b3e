"""What is measured of the decoder-training operators: rotary positions, the gated linear layer, distillation from a
teacher's top logits and the clipped policy loss, each with its gradient.

``run`` computes a case either in plain torch operations (``own`` false) or through the library's public entry points
(``own`` true); ``exact`` computes it again in 64 bits from the definitions.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

DEV = "cuda"
BIG_LOGITS = 8192 * 32000          # most logits of a loss case
BIG_ROTARY = 3 * 32771 * 12 * 80   # most values of a rotary case
BIG_GATED = 8192 * 4096 * 4096     # most ndat * xvec * yvec of a gated case


def listed():
    return [
        # one token of a sequence that is already long: q of the attention configuration (8 heads of 64); latency
        dict(name="rotary token", op="rotary", nbat=1, ntimes=1, nhead=8, npiece=64, nrot=64, half=True, parts=False,
             backward=False, first=100003),
        # the attention configuration, 32 x 512 tokens, neighbouring values form the pairs
        dict(name="rotary batch", op="rotary", nbat=32, ntimes=512, nhead=8, npiece=64, nrot=64, half=False, parts=False,
             backward=False, first=0),
        # gradient on long sequences, half of an 80-wide head rotated, frequencies scaled by parts
        dict(name="rotary long backward", op="rotary", nbat=3, ntimes=32771, nhead=12, npiece=80, nrot=40, half=True,
             parts=True, backward=True, first=17),
        # serving: one token through a 4096 x 4096 layer, bound by the weights
        dict(name="gated token", op="gated", ndat=1, xvec=4096, yvec=4096, act="swish", train=False, bias=False),
        # serving a batch of sequences, one token each
        dict(name="gated tokens", op="gated", ndat=48, xvec=4096, yvec=4096, act="swish", train=False, bias=False),
        # a small model's training step, odd sizes and biases
        dict(name="gated small step", op="gated", ndat=391, xvec=512, yvec=1365, act="gelu", train=True, bias=True),
        # the Linear step configuration (8192 tokens, 4096 wide) as a gated layer: forward and all gradients
        dict(name="gated step", op="gated", ndat=8192, xvec=4096, yvec=4096, act="swish", train=True, bias=False),
        # one row: the call's latency
        dict(name="distill row", op="distill", nrow=1, ncol=32000, ntop=32, mode="step", used=1.0),
        # an odd vocabulary; loss and gradient as two calls, as an autograd graph makes them; a quarter of the rows is padding
        dict(name="distill two calls", op="distill", nrow=1021, ncol=50257, ntop=64, mode="calls", used=0.75),
        # a large batch, loss and gradient in one call
        dict(name="distill step", op="distill", nrow=8192, ncol=32000, ntop=64, mode="step", used=1.0),
        # log-probabilities and loss of a handful of tokens
        dict(name="policy rows", op="policy", nrow=7, ncol=32000, mode="loss", used=1.0, ref=True),
        # a training batch with padding, odd vocabulary
        dict(name="policy step", op="policy", nrow=4096, ncol=50257, mode="step", used=0.9, ref=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "gated", "distill", "policy"])
    if op == "rotary":
        nhead, npiece = rng.randint(1, 24), 2 * rng.randint(8, 64)
        nrot = npiece if rng.random() < 0.5 else 2 * rng.randint(1, npiece // 2)
        nbat = _log_int(rng, 1, 64)
        ntimes = _log_int(rng, 1, max(1, min(65536, BIG_ROTARY // (nbat * nhead * npiece))))
        return dict(op=op, nbat=nbat, ntimes=ntimes, nhead=nhead, npiece=npiece, nrot=nrot, half=rng.random() < 0.5,
                    parts=rng.random() < 0.5, backward=rng.random() < 0.5, first=rng.randint(0, 200000))
    if op == "gated":
        xvec, yvec = _log_int(rng, 64, 4096), _log_int(rng, 64, 4096)
        ndat = _log_int(rng, 1, max(1, min(8192, BIG_GATED // (xvec * yvec))))
        return dict(op=op, ndat=ndat, xvec=xvec, yvec=yvec, act=rng.choice(["swish", "gelu", "relu", "sigmoid"]),
                    train=rng.random() < 0.6, bias=rng.random() < 0.5)
    ncol = _log_int(rng, 97, 128256)
    nrow = _log_int(rng, 1, max(1, min(8192, BIG_LOGITS // ncol)))
    used = rng.choice([1.0, 0.9, 0.5])
    if op == "distill":
        return dict(op=op, nrow=nrow, ncol=ncol, ntop=min(ncol, _log_int(rng, 1, 256)),
                    mode=rng.choice(["loss", "calls", "step"]), used=used)
    return dict(op=op, nrow=nrow, ncol=ncol, mode=rng.choice(["loss", "calls", "step"]), used=used, ref=rng.random() < 0.7)


# ---- inputs ----------------------------------------------------------------------------------------
def _frequencies(nrot, parts):
    """Radians per position of every pair, 64 bits; `parts`: long wavelengths stretched eightfold, short ones kept."""
    i = torch.arange(nrot // 2, device=DEV, dtype=torch.float64)
    f = torch.exp(i * (-2.0 / nrot * math.log(10000.0)))
    if parts:
        keep = ((f * (4096 / (2 * math.pi)) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * (keep + (1 - keep) / 8.0)
    return f


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device=DEV, generator=gen)  # noqa: E731
    empty = lambda *shape: torch.empty(shape, device=DEV)                  # noqa: E731
    scalar = lambda v: torch.tensor([v], device=DEV)                       # noqa: E731
    s = dict(case)
    if case["op"] == "rotary":
        nbat, ntimes, nvec = case["nbat"], case["ntimes"], case["nhead"] * case["npiece"]
        s["x"] = normal(nbat, ntimes, nvec)
        s["freq"] = _frequencies(case["nrot"], case["parts"])
        # every sequence of the batch begins at a place of its own
        start = case["first"] + torch.randint(0, 1000, (nbat, 1), device=DEV, generator=gen)
        s["pos"] = start + torch.arange(ntimes, device=DEV)
        s["scale"] = scalar(0.1 * math.log(8.0) + 1.0) if case["parts"] else None
        s["y"] = empty(nbat, ntimes, nvec)
        return s
    if case["op"] == "gated":
        m, k, f = case["ndat"], case["xvec"], case["yvec"]
        s["x"] = normal(m, k)
        s["wg"], s["wu"] = normal(f, k) / math.sqrt(k), normal(f, k) / math.sqrt(k)
        s["bg"], s["bu"] = (normal(f), normal(f)) if case["bias"] else (None, None)
        s["h"] = empty(m, f)
        if case["train"]:
            s["gh"] = normal(m, f)
            s["g"], s["u"], s["gg"], s["gu"] = empty(m, f), empty(m, f), empty(m, f), empty(m, f)
            s["gx"], s["gwg"], s["gwu"] = empty(m, k), empty(f, k), empty(f, k)
        return s
    n, c = case["nrow"], case["ncol"]
    s["x"] = normal(n, c) * 2.5
    s["y"], s["stat"] = empty(n), empty(n, 3)
    if case["mode"] != "loss":
        s["gx"] = empty(n, c)
    live = torch.rand(n, device=DEV, generator=gen) < case["used"]
    s["gy"] = live.float() / n                  # the mean over the batch, as its gradient
    if case["op"] == "distill":
        k = case["ntop"]
        s["temp"] = scalar(2.0)
        # ids without repetition in a row: a random start, then even steps around the vocabulary
        start = torch.randint(0, c, (n, 1), device=DEV, generator=gen)
        s["idx"] = ((start + torch.arange(k, device=DEV) * max(1, c // k)) % c).int()
        s["t"] = (normal(n, k) * 3).sort(dim=1, descending=True).values + 8
        tail = torch.randint(max(1, k // 2), k + 1, (n, 1), device=DEV, generator=gen)
        s["idx"][torch.arange(k, device=DEV) >= tail] = -1      # rows with fewer entries than the table is wide
        s["idx"][~live] = -1
        return s
    s["temp"] = scalar(1.0)
    z = torch.randint(0, c, (n,), device=DEV, generator=gen)
    s["x"][torch.arange(n, device=DEV), z] += 8                 # sampled tokens are likely ones
    now = _log_prob(s["x"], z, s["temp"])[0]
    s["old"] = (now + 0.15 * normal(n)).float()
    s["ref"] = (now + 0.3 * normal(n)).float() if case["ref"] else None
    s["adv"] = normal(n)
    s["z"] = torch.where(live, z, -1).int()
    s["low"], s["high"], s["beta"] = scalar(0.2), scalar(0.25), scalar(0.04)
    s["logp"] = empty(n)
    return s


# ---- plain forms -----------------------------------------------------------------------------------
def _rotary(s):
    x = s["x"].view(s["nbat"], s["ntimes"], s["nhead"], s["npiece"])
    turn = s["pos"].double()[..., None] * s["freq"]             # angles of far positions: 64 bits
    cos, sin = torch.cos(turn).float()[:, :, None], torch.sin(turn).float()[:, :, None]
    if s["backward"]:
        sin = -sin
    if s["scale"] is not None:
        cos, sin = cos * s["scale"], sin * s["scale"]
    r = s["nrot"]
    a, b = (x[..., : r // 2], x[..., r // 2: r]) if s["half"] else (x[..., 0:r:2], x[..., 1:r:2])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([p, q], -1) if s["half"] else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1).view_as(s["x"])


def _act(name, v):
    """The activation and its slope."""
    if name == "relu":
        return v * (v > 0), (v > 0).float()
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))
        return v * cdf, cdf + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi))
    sig = 1 / (1 + torch.exp(-v))
    return (sig, sig * (1 - sig)) if name == "sigmoid" else (v * sig, sig * (1 + v * (1 - sig)))


def _gated(s):
    g, u = s["x"] @ s["wg"].T, s["x"] @ s["wu"].T
    if s["bias"]:
        g, u = g + s["bg"], u + s["bu"]
    a, slope = _act(s["act"], g)
    if not s["train"]:
        return a * u
    gg, gu = s["gh"] * u * slope, s["gh"] * a
    return a * u, gg @ s["wg"] + gu @ s["wu"], gg.T @ s["x"], gu.T @ s["x"], gg, gu


def _softmax(x, temp):
    """Exponentials against the row maximum, that maximum, and their sum in 64 bits."""
    top = x.amax(-1, keepdim=True)
    e = torch.exp((x - top) / temp)
    return e, top, e.sum(-1, dtype=torch.float64)


def _log_prob(x, z, temp):
    e, top, total = _softmax(x, temp)
    at = x.gather(1, z[:, None].long().clamp(min=0))
    return (at - top)[:, 0].double() / temp - torch.log(total), e, total


def _distill(s):
    x, t, temp = s["x"], s["t"], s["temp"]
    used = s["idx"] >= 0
    at = s["idx"].long().clamp(min=0)
    live = used.any(-1)
    t = torch.where(used, t, -math.inf) / temp
    w = torch.where(used, torch.exp(t - torch.where(live, t.amax(-1), 0.0)[:, None]), 0.0)
    p = w / torch.where(live, w.sum(-1), 1.0)[:, None]
    e, top, total = _softmax(x, temp)
    logq = (x.gather(1, at) - top).double() / temp - torch.log(total)[:, None]
    logp = torch.log(torch.where(p > 0, p, 1.0).double())
    y = (temp.double() ** 2 * torch.where(p > 0, p * (logp - logq), 0.0).sum(-1)).float()
    if s["mode"] == "loss":
        return y
    gx = e * (live / total).float()[:, None]
    gx.scatter_add_(1, at, -p)
    return y, gx * (s["gy"] * temp)[:, None]


def _policy(s):
    logp, e, total = _log_prob(s["x"], s["z"], s["temp"])
    live = s["z"] >= 0
    adv, ratio = s["adv"].double(), torch.exp(logp - s["old"])
    bound = torch.minimum(torch.maximum(ratio, 1 - s["low"].double()), 1 + s["high"].double())
    free = ratio * adv <= bound * adv
    y, slope = -torch.where(free, ratio * adv, bound * adv), -adv * ratio * free
    if s["ref"] is not None:
        d = s["ref"] - logp
        y, slope = y + s["beta"] * (torch.exp(d) - d - 1), slope + s["beta"] * (1 - torch.exp(d))
    y, logp = torch.where(live, y, 0.0).float(), torch.where(live, logp, 0.0).float()
    if s["mode"] == "loss":
        return y, logp
    c = torch.where(live, slope, 0.0) * s["gy"] / s["temp"]
    gx = e * (-c / total).float()[:, None]
    gx.scatter_add_(1, s["z"].long().clamp(min=0)[:, None], c.float()[:, None])
    return y, logp, gx


# ---- the library's entry points ----------------------------------------------------------------------
_vm = None


def _vmath():
    global _vm
    if _vm is None:
        _vm = importlib.import_module("deep-learning-framework_b200").vmath
    return _vm


def _own_rotary(s):
    vm = _vmath()
    call = vm.rotary_backward if s["backward"] else vm.rotary
    call(0, s["y"], s["x"], s["freq"], s["pos"], 0, s["nbat"], s["ntimes"], s["nhead"], s["npiece"], s["nrot"],
         "half" if s["half"] else "interleaved", s["scale"])
    return s["y"]


def _own_gated(s):
    vm = _vmath()
    f, m, k = s["yvec"], s["ndat"], s["xvec"]
    if not s["train"]:
        vm.gated_linear_forward(0, s["h"], None, None, s["wg"], s["wu"], s["x"], s["bg"], s["bu"], f, m, k, s["act"])
        return s["h"]
    vm.gated_linear_forward(0, s["h"], s["g"], s["u"], s["wg"], s["wu"], s["x"], s["bg"], s["bu"], f, m, k, s["act"])
    vm.gated_linear_backward(0, s["gx"], s["gwg"], s["gwu"], s["gg"], s["gu"], s["gh"], s["g"], s["u"], s["wg"], s["wu"],
                             s["x"], f, m, k, s["act"])
    return s["h"], s["gx"], s["gwg"], s["gwu"], s["gg"], s["gu"]


def _own_distill(s):
    vm = _vmath()
    n, c, k = s["nrow"], s["ncol"], s["ntop"]
    if s["mode"] == "step":
        vm.softmax_top_distill_step(0, s["y"], s["gx"], s["gy"], s["x"], s["idx"], s["t"], n, c, k, s["temp"])
        return s["y"], s["gx"]
    vm.softmax_top_distill(0, s["y"], s["stat"], s["x"], s["idx"], s["t"], n, c, k, s["temp"])
    if s["mode"] == "loss":
        return s["y"]
    vm.softmax_top_distill_backward_x(0, s["gx"], s["gy"], s["x"], s["stat"], s["idx"], s["t"], n, c, k, s["temp"])
    return s["y"], s["gx"]


def _own_policy(s):
    vm = _vmath()
    n, c = s["nrow"], s["ncol"]
    if s["mode"] == "step":
        vm.softmax_policy_loss_step(0, s["y"], s["logp"], s["gx"], s["gy"], s["x"], s["z"], s["old"], s["ref"], s["adv"],
                                    n, c, s["low"], s["high"], s["beta"], s["temp"])
        return s["y"], s["logp"], s["gx"]
    vm.softmax_policy_loss(0, s["y"], s["logp"], s["stat"], s["x"], s["z"], s["old"], s["ref"], s["adv"], n, c, s["low"],
                           s["high"], s["beta"], s["temp"])
    if s["mode"] == "loss":
        return s["y"], s["logp"]
    vm.softmax_policy_loss_backward_x(0, s["gx"], s["gy"], s["x"], s["stat"], s["z"], n, c, s["temp"])
    return s["y"], s["logp"], s["gx"]


def run(state):
    if own:
        return {"rotary": _own_rotary, "gated": _own_gated, "distill": _own_distill, "policy": _own_policy}[state["op"]](state)
    return {"rotary": _rotary, "gated": _gated, "distill": _distill, "policy": _policy}[state["op"]](state)


def work(case):
    if case["op"] == "rotary":
        tokens = case["nbat"] * case["ntimes"]
        n = tokens * case["nhead"] * case["npiece"]
        return {"bytes": 8 * n + 8 * tokens + 4 * case["nrot"], "flops": 3 * tokens * case["nhead"] * case["nrot"]}
    if case["op"] == "gated":
        m, k, f = case["ndat"], case["xvec"], case["yvec"]
        once = m * k + 2 * k * f + m * f
        if not case["train"]:
            return {"bytes": 4 * once, "flops": 4 * m * k * f}
        # read x, both weights and the output's gradient; write h, the two pre-activation gradients and three gradients
        return {"bytes": 4 * (2 * once + 2 * m * f), "flops": 12 * m * k * f}
    n, c = case["nrow"], case["ncol"]
    table = 8 * n * case["ntop"] if case["op"] == "distill" else 16 * n
    both = case["mode"] != "loss"
    return {"bytes": (8 if both else 4) * n * c + table + 8 * n, "flops": (6 if both else 4) * n * c}


# ---- 64 bits, from the definitions -------------------------------------------------------------------
def _exact_rotary(s):
    x = s["x"].double().view(s["nbat"], s["ntimes"], s["nhead"], s["npiece"])
    r = s["nrot"]
    head = x[..., :r]
    pair = head.unflatten(-1, (2, r // 2)).transpose(-1, -2) if s["half"] else head.unflatten(-1, (r // 2, 2))
    number = torch.view_as_complex(pair.contiguous())
    angle = s["pos"].double()[:, :, None, None] * s["freq"] * (-1.0 if s["backward"] else 1.0)
    size = torch.ones_like(angle) if s["scale"] is None else torch.full_like(angle, float(s["scale"]))
    out = torch.view_as_real(number * torch.polar(size, angle))
    out = (out.transpose(-1, -2) if s["half"] else out).flatten(-2)
    return torch.cat([out, x[..., r:]], -1).reshape(s["x"].shape)


def _exact_gated(s):
    names = {"relu": torch.relu, "sigmoid": torch.sigmoid, "swish": torch.nn.functional.silu,
             "gelu": torch.nn.functional.gelu}
    x, wg, wu = (s[n].double().requires_grad_() for n in ("x", "wg", "wu"))
    g, u = torch.einsum("mk,fk->mf", x, wg), torch.einsum("mk,fk->mf", x, wu)
    if s["bias"]:
        g, u = g + s["bg"].double(), u + s["bu"].double()
    h = names[s["act"]](g) * u
    if not s["train"]:
        return h.detach()
    grads = torch.autograd.grad(h, (x, wg, wu, g, u), s["gh"].double())
    return (h.detach(), *grads)


def _exact_distill(s):
    ys, gs = [], []
    for rows in torch.arange(s["nrow"], device=DEV).split(2048):
        x = s["x"][rows].double().requires_grad_()
        idx, t, temp = s["idx"][rows].long(), s["t"][rows].double(), float(s["temp"])
        live = (idx >= 0).any(-1)
        t = torch.where((idx >= 0) | ~live[:, None], t / temp, -math.inf)
        log_p = t - torch.logsumexp(t, -1, keepdim=True)
        log_q = torch.log_softmax(x / temp, -1).gather(1, idx.clamp(min=0))
        p = torch.exp(log_p)
        term = p * (torch.where(p > 0, log_p, 0.0) - log_q)
        y = torch.where(live, temp * temp * term.sum(-1), 0.0)
        ys.append(y.detach())
        if s["mode"] != "loss":
            gs.append(torch.autograd.grad(y, x, s["gy"][rows].double())[0])
    return torch.cat(ys) if s["mode"] == "loss" else (torch.cat(ys), torch.cat(gs))


def _exact_policy(s):
    ys, ls, gs = [], [], []
    for rows in torch.arange(s["nrow"], device=DEV).split(1024):
        x = s["x"][rows].double().requires_grad_()
        z, live = s["z"][rows].long(), s["z"][rows] >= 0
        logp = torch.log_softmax(x / float(s["temp"]), -1).gather(1, z.clamp(min=0)[:, None])[:, 0]
        ratio, adv = torch.exp(logp - s["old"][rows].double()), s["adv"][rows].double()
        y = -torch.minimum(ratio * adv, ratio.clamp(1 - float(s["low"]), 1 + float(s["high"])) * adv)
        if s["ref"] is not None:
            gap = s["ref"][rows].double() - logp
            y = y + float(s["beta"]) * (torch.expm1(gap) - gap)
        y = torch.where(live, y, 0.0)
        ys.append(y.detach())
        ls.append(torch.where(live, logp, 0.0).detach())
        if s["mode"] != "loss":
            gs.append(torch.autograd.grad(y, x, s["gy"][rows].double())[0])
    return (torch.cat(ys), torch.cat(ls)) if s["mode"] == "loss" else (torch.cat(ys), torch.cat(ls), torch.cat(gs))


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "gated": _exact_gated, "distill": _exact_distill, "policy": _exact_policy}[case["op"]](s)
