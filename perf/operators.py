"""Operators of recurrent on-policy training, timed and compared on the GPU: the gated linear recurrence that gives a
policy its memory (whole sequences with their gradients, and one step of a rollout), the advantages of an episode, the
clipped policy loss with its KL term and its gradients, and the sampling of a Gaussian policy's actions.

`own` False: the plain forms below, elementary torch operations.  `own` True: marl_amd.recurrence / marl_amd.policy_loss."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # 64 environments x 30 agents, an episode of 200 steps, hidden width 256: one training pass of a policy's memory
        dict(name="scan_train_episode", op="scan", T=200, B=1920, D=256, dtype="float32", batch_first=False, resets=False, lengths=False, h0=True, train=True),
        # bf16 training on whole and broken-off episodes, stored sequence by sequence, several episodes to a row
        dict(name="scan_train_ragged_bf16", op="scan", T=200, B=491, D=128, dtype="bfloat16", batch_first=True, resets=True, lengths=True, h0=True, train=True),
        # a few long recordings, an odd width: little to run side by side but the time axis
        dict(name="scan_train_long", op="scan", T=20011, B=3, D=61, dtype="float32", batch_first=False, resets=True, lengths=False, h0=False, train=True),
        # one environment of 30 agents: the memory after the first steps of an evaluation, no gradients
        dict(name="scan_eval_small", op="scan", T=37, B=30, D=64, dtype="float32", batch_first=False, resets=False, lengths=False, h0=True, train=False),
        # a rollout's step: 4096 environments x 30 agents, width 256, some environments starting over
        dict(name="step_rollout", op="step", B=122880, D=256, dtype="float32", resets=True),
        # one environment's step: latency
        dict(name="step_single_env", op="step", B=30, D=64, dtype="float32", resets=False),
        # advantages of an episode of 4096 environments x 30 agents, with what the loss needs to normalise them
        dict(name="advantages_episode", op="advantages", T=200, E=4096, n=30, dones=False, lengths=False, moments=True),
        # seven environments that end at different times, an odd number of steps
        dict(name="advantages_ragged_small", op="advantages", T=333, E=7, n=13, dones=True, lengths=True, moments=False),
        # the policy loss over that whole episode: 24.6 million rows, actions as the replay stores them
        dict(name="loss_episode", op="loss", B=819200, n=30, A=2, dtype="float32", shared_std=True, mask=False, ref=False, moments=True),
        # a minibatch of 2048 rows, bf16 network, a deviation for each row, padded rows, a reference policy
        dict(name="loss_minibatch_bf16", op="loss", B=1, n=2048, A=2, dtype="bfloat16", shared_std=False, mask=True, ref=True, moments=False),
        # a rollout's actions and their log-probabilities, written where the replay keeps them
        dict(name="act_rollout", op="act", B=4096, n=30, A=2, dtype="float32", shared_std=True),
        # one environment's actions: latency
        dict(name="act_single_env", op="act", B=1, n=30, A=2, dtype="float32", shared_std=True),
    ]


def _span(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "step", "advantages", "loss", "loss", "act"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    dtype = rng.choice(["float32", "float32", "bfloat16"])
    if op == "scan":
        T, D = _span(rng, 1, 20011), _span(rng, 8, 256)
        most = 98304000 * 8 // (max(1, math.ceil(math.log2(max(2, T)))) * T * D)       # (the plain form's passes grow with log T)
        B = _span(rng, 1, max(1, min(1920, most)))
        return dict(op=op, T=T, B=B, D=D, dtype=dtype, batch_first=flag(), resets=flag(), lengths=flag(), h0=flag(), train=rng.random() < 0.75)
    if op == "step":
        return dict(op=op, B=_span(rng, 1, 122880), D=_span(rng, 8, 256), dtype=dtype, resets=flag())
    if op == "advantages":
        T, n = _span(rng, 1, 2000), _span(rng, 1, 64)
        return dict(op=op, T=T, E=_span(rng, 1, max(1, min(4096, 24576000 // (T * n)))), n=n, dones=flag(), lengths=flag(), moments=flag())
    if op == "loss":
        n, A = _span(rng, 1, 2048), rng.choice([1, 2, 2, 3, 4, 7])
        return dict(op=op, B=_span(rng, 1, max(1, 24576000 // (n * A))), n=n, A=A, dtype=dtype, shared_std=flag(), mask=flag(), ref=flag(), moments=flag())
    n = _span(rng, 1, 1024)
    return dict(op=op, B=_span(rng, 1, max(1, 122880 // n)), n=n, A=rng.choice([1, 2, 2, 3, 4, 7]), dtype=dtype, shared_std=flag())


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    rand = lambda *s: torch.rand(*s, device=DEV, generator=gen)  # noqa: E731
    s = dict(case)
    op = case["op"]
    if op in ("scan", "step"):
        dt = TYPES[case["dtype"]]
        B, D = case["B"], case["D"]
        lead = (B,) if op == "step" else (B, case["T"]) if case["batch_first"] else (case["T"], B)
        s["gate"] = (randn(*lead, D) + 2.0).to(dt)                       # a memory of about ten steps, as a trained gate keeps
        s["x"] = randn(*lead, D).to(dt)
        s["h0"] = randn(B, D) if op == "step" or case["h0"] else None
        if op == "step":
            s["reset"] = rand(B) < 0.005 if case["resets"] else None
            s["out"] = torch.empty(B, D, device=DEV, dtype=dt)           # a rollout hands the same buffer every step
            return s
        s["reset"] = rand(*lead) < 0.005 if case["resets"] else None     # (episodes of about 200 steps)
        s["len"] = torch.randint(0, case["T"] + 1, (B,), device=DEV, generator=gen, dtype=torch.int32) if case["lengths"] else None
        if case["train"]:
            s["dh"] = randn(*lead, D).to(dt)
            s["dlast"] = randn(B, D)
            for k in ("gate", "x", "h0"):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    if op == "advantages":
        T, E, n = case["T"], case["E"], case["n"]
        s["rewards"] = (rand(T, E, n) < 0.3).float()                     # the environment's binary reward
        s["values"] = randn(T + 1, E, n) * 0.5 + 4.0
        s["done"] = rand(T, E, n) < 0.01 if case["dones"] else None
        s["len"] = torch.randint(0, T + 1, (E,), device=DEV, generator=gen, dtype=torch.int32) if case["lengths"] else None
        return s
    B, n, A = case["B"], case["n"], case["A"]
    dt = TYPES[case["dtype"]]
    s["mean"] = torch.tanh(randn(B, n, A)).to(dt)
    std = randn(A) * 0.2 - 0.7 if case["shared_std"] else randn(B, n, A) * 0.2 - 0.7
    s["log_std"] = std.to(dt)
    noise = randn(B, n, A)
    if op == "act":
        s["noise"] = noise
        s["ring"] = torch.empty(B, A, n, device=DEV)                     # agents contiguous, as the environment reads them
        s["log_pi"] = torch.empty(B, n, device=DEV)
        return s
    std = s["log_std"].float()
    rows = s["mean"].float() + 0.1 * randn(B, n, A) + noise * std.exp()  # drawn by a policy some updates older
    s["ring"] = rows.transpose(1, 2).contiguous()
    z = ((rows - s["mean"].float()) * (-std).exp())
    now = (-0.5 * z * z - std - 0.5 * math.log(2 * math.pi)).sum(-1)
    s["log_pi_old"] = now + 0.2 * randn(B, n)
    s["log_pi_ref"] = now + 0.2 * randn(B, n) if case["ref"] else None
    s["adv"] = randn(B, n) * 2.0 + 0.5
    s["mask"] = rand(B, n) < 0.9 if case["mask"] else None
    s["moments"] = torch.stack([s["adv"].mean(), 1.0 / s["adv"].std()]) if case["moments"] else None
    s["mean"].requires_grad_()
    s["log_std"].requires_grad_()
    return s


CLIP, KL, ENTROPY, GAMMA, LAMBDA = 0.2, 0.05, 0.01, 0.95, 0.95


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from marl_amd import policy_loss, recurrence
    op = s["op"]
    if op == "scan":
        h, last = recurrence.gated_scan(s["gate"], s["x"], s["h0"], resets=s["reset"], lengths=s["len"], batch_first=s["batch_first"])
        if not s["train"]:
            return h, last
        leaves = [s[k] for k in ("gate", "x", "h0") if s[k] is not None]
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), leaves, (s["dh"], s["dlast"]))
    if op == "step":
        return recurrence.gated_scan_step(s["gate"], s["x"], s["h0"], reset=s["reset"], out=s["out"]), s["h0"]
    if op == "advantages":
        return recurrence.advantages(s["rewards"], s["values"], dones=s["done"], lengths=s["len"], gamma=GAMMA, lam=LAMBDA, moments=s["moments"])
    actions = s["ring"].transpose(1, 2)
    if op == "act":
        return policy_loss.gaussian_act(s["mean"], s["log_std"], s["noise"], actions=actions, log_pi=s["log_pi"])
    loss, stats = policy_loss.clipped_policy_loss(s["mean"], s["log_std"], actions, s["log_pi_old"], s["adv"], log_pi_ref=s["log_pi_ref"],
                                                  mask=s["mask"], adv_moments=s["moments"], clip=CLIP, kl_coef=KL, entropy_coef=ENTROPY)
    return (loss.detach(), stats) + torch.autograd.grad(loss, (s["mean"], s["log_std"]))


# ---- plain forms ------------------------------------------------------------------------------

def _affine_scan(a, u):
    """y_t = a_t y_{t-1} + u_t along the first axis, y_{-1} = 0: doubling, log2(T) passes."""
    s = 1
    while s < u.shape[0]:
        u = torch.cat((u[:s], u[s:] + a[s:] * u[:-s]))
        a = torch.cat((a[:s], a[s:] * a[:-s]))
        s *= 2
    return u


def _plain(s):
    return {"scan": _plain_scan, "step": _plain_step, "advantages": _plain_advantages, "loss": _plain_loss, "act": _plain_act}[s["op"]](s)


@torch.no_grad()
def _plain_scan(s):
    first = lambda t: t.transpose(0, 1) if s["batch_first"] else t  # noqa: E731
    dt = s["gate"].dtype
    g, x = first(s["gate"]).float(), first(s["x"]).float()
    T, B, D = g.shape
    h0 = torch.zeros(B, D, device=DEV) if s["h0"] is None else s["h0"]
    a, b = torch.sigmoid(g), torch.sigmoid(-g)
    keep = torch.ones(T, B, 1, device=DEV, dtype=torch.bool) if s["reset"] is None else ~first(s["reset"]).unsqueeze(-1)
    valid = torch.ones(T, B, 1, device=DEV, dtype=torch.bool)
    if s["len"] is not None:
        valid = (torch.arange(T, device=DEV).unsqueeze(1) < s["len"]).unsqueeze(-1)
    zero, one = torch.zeros((), device=DEV), torch.ones((), device=DEV)
    carry = torch.where(valid, torch.where(keep, a, zero), one)          # what is left of the state before
    u = torch.where(valid, b * x, zero)
    u = torch.cat(((u[:1] + carry[:1] * h0), u[1:]))
    h = _affine_scan(carry, u)
    out = first(torch.where(valid, h, zero)).to(dt).contiguous()
    if not s["train"]:
        return out, h[-1]
    dh = torch.where(valid, first(s["dh"]).float(), zero)
    dh = torch.cat((dh[:-1], dh[-1:] + s["dlast"]))
    after = torch.cat((carry[1:], torch.zeros_like(carry[:1])))          # dL/dh_t = dh_t + carry_{t+1} dL/dh_{t+1}
    G = _affine_scan(after.flip(0), dh.flip(0)).flip(0)
    before = torch.where(keep, torch.cat((h0.unsqueeze(0), h[:-1])), zero)
    dx = first(torch.where(valid, G * b, zero)).to(dt).contiguous()
    dgate = first(torch.where(valid, G * (before - x) * a * b, zero)).to(dt).contiguous()
    return (out, h[-1], dgate, dx) + (() if s["h0"] is None else (carry[0] * G[0],))


@torch.no_grad()
def _plain_step(s):
    g, x, h = s["gate"].float(), s["x"].float(), s["h0"]
    before = h if s["reset"] is None else torch.where(s["reset"].unsqueeze(-1), torch.zeros((), device=DEV), h)
    h.copy_(torch.sigmoid(g) * before + torch.sigmoid(-g) * x)
    s["out"].copy_(h)
    return s["out"], h


@torch.no_grad()
def _plain_advantages(s):
    r, v = s["rewards"], s["values"]
    T, E, n = r.shape
    zero, one = torch.zeros((), device=DEV), torch.ones((), device=DEV)
    valid = torch.ones(T, E, 1, device=DEV, dtype=torch.bool)
    if s["len"] is not None:
        valid = (torch.arange(T, device=DEV).unsqueeze(1) < s["len"]).unsqueeze(-1)
    go = one.expand(T, E, n) if s["done"] is None else torch.where(s["done"], zero, one)
    delta = torch.where(valid, r + GAMMA * torch.where(go > 0, v[1:], zero) - v[:-1], zero)
    adv = _affine_scan((GAMMA * LAMBDA * go).flip(0), delta.flip(0)).flip(0)
    adv = torch.where(valid, adv, zero)
    ret = torch.where(valid, adv + v[:-1], zero)
    if not s["moments"]:
        return adv, ret
    count = valid.expand(T, E, n).sum().double().clamp_min(1.0)
    mean = adv.double().sum() / count
    var = torch.where(valid, (adv.double() - mean) ** 2, torch.zeros((), device=DEV, dtype=torch.float64)).sum() / count
    return adv, ret, torch.stack([mean, 1.0 / (var.sqrt() + 1e-8)]).float()


@torch.no_grad()
def _plain_act(s):
    mean, std = s["mean"].float(), s["log_std"].float().expand(s["mean"].shape)
    act = mean + std.exp() * s["noise"]
    z = (act - mean).double() * (-std.double()).exp()
    s["ring"].copy_(act.transpose(1, 2))
    s["log_pi"].copy_((-0.5 * z * z - std.double() - 0.5 * math.log(2 * math.pi)).sum(-1))
    return s["ring"].transpose(1, 2), s["log_pi"]


@torch.no_grad()
def _plain_loss(s):
    # (64 bits: a ratio next to the clipping border, and the KL estimate of two nearly equal policies)
    mean, std = s["mean"].double(), s["log_std"].double()
    z = (s["ring"].transpose(1, 2).double() - mean) * (-std).exp()
    log_pi = (-0.5 * z * z - std - 0.5 * math.log(2 * math.pi)).sum(-1)
    adv = s["adv"].double()
    if s["moments"] is not None:
        m = s["moments"].double()
        adv = (adv - m[0]) * m[1]
    ref = s["log_pi_old"] if s["log_pi_ref"] is None else s["log_pi_ref"]
    ratio = (log_pi - s["log_pi_old"].double()).exp()
    off = ref.double() - log_pi
    kl = torch.expm1(off) - off
    entropy = (std + 0.5 * math.log(2 * math.pi * math.e)).expand(mean.shape).sum(-1)
    valid = torch.ones_like(ratio, dtype=torch.bool) if s["mask"] is None else s["mask"]
    zero = torch.zeros((), device=DEV, dtype=torch.float64)
    count = valid.sum().double().clamp_min(1.0)
    lo, hi = 1.0 - CLIP, 1.0 + CLIP
    gain = torch.minimum(ratio * adv, ratio.clamp(lo, hi) * adv)
    cut = ((adv > 0) & (ratio > hi)) | ((adv < 0) & (ratio < lo))
    mid = lambda t: torch.where(valid, t, zero).sum() / count  # noqa: E731
    gain, klm, ent, cutm, rat = mid(gain), mid(kl), mid(entropy), mid(cut.double()), mid(ratio)
    loss = -gain + KL * klm - ENTROPY * ent
    stats = torch.stack([gain, klm, ent, cutm, rat, valid.sum().double()]).float()
    w = torch.where(valid, 1.0 / count, zero)
    dlog = torch.where(valid, w * (torch.where(cut, zero, -ratio * adv) - KL * torch.expm1(off)), zero).unsqueeze(-1)
    dmean = torch.where(valid.unsqueeze(-1), dlog * z * (-std).exp(), zero)
    dstd = torch.where(valid.unsqueeze(-1), dlog * (z * z - 1.0) - ENTROPY * w.unsqueeze(-1), zero)
    if s["shared_std"]:
        dstd = dstd.sum((0, 1))
    return loss.float(), stats, dmean.to(s["mean"].dtype), dstd.to(s["log_std"].dtype)


# ---- 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"scan": _exact_scan, "step": _exact_step, "advantages": _exact_advantages, "loss": _exact_loss, "act": _exact_act}[case["op"]](s)


def _exact_scan(s):
    """Step by step through time, and back."""
    dim = 1 if s["batch_first"] else 0
    g, x = s["gate"].double(), s["x"].double()
    T, D = g.shape[dim], g.shape[2]
    B = g.shape[1 - dim]
    a = 1.0 / (1.0 + torch.exp(-g))
    h = torch.zeros(B, D, device=DEV, dtype=torch.float64) if s["h0"] is None else s["h0"].double()
    states, outs = [h], []
    on = lambda t: None if s["len"] is None else (s["len"] > t).unsqueeze(1)  # noqa: E731
    for t in range(T):
        at = a.select(dim, t)
        kept = h if s["reset"] is None else h.masked_fill(s["reset"].select(dim, t).unsqueeze(1), 0.0)
        new = at * kept + (1.0 - at) * x.select(dim, t)
        if on(t) is not None:
            outs.append(new * on(t))
            h = torch.where(on(t), new, h)
        else:
            outs.append(new)
            h = new
        states.append(h)
    out = torch.stack(outs, dim)
    if not s["train"]:
        return out, h
    G = s["dlast"].double()                                             # dL/dh behind the last step
    dgate, dx = torch.zeros_like(g), torch.zeros_like(x)
    for t in range(T - 1, -1, -1):
        at, xt, dt = a.select(dim, t), x.select(dim, t), s["dh"].select(dim, t).double()
        kept = states[t] if s["reset"] is None else states[t].masked_fill(s["reset"].select(dim, t).unsqueeze(1), 0.0)
        here = G + dt
        dg, du = here * (kept - xt) * at * (1.0 - at), here * (1.0 - at)
        back = here * at
        if s["reset"] is not None:
            back = back.masked_fill(s["reset"].select(dim, t).unsqueeze(1), 0.0)
        if on(t) is not None:
            dg, du, back = dg * on(t), du * on(t), torch.where(on(t), back, G)
        dgate.select(dim, t).copy_(dg)
        dx.select(dim, t).copy_(du)
        G = back
    return (out, h, dgate, dx) + (() if s["h0"] is None else (G,))


def _exact_step(s):
    a = 1.0 / (1.0 + torch.exp(-s["gate"].double()))
    h = s["h0"].double()
    if s["reset"] is not None:
        h = h * (~s["reset"]).double().unsqueeze(1)
    h = h * a + s["x"].double() * (1.0 - a)
    return h, h


def _exact_advantages(s):
    r, v = s["rewards"].double(), s["values"].double()
    adv, ret, run_ = torch.zeros_like(r), torch.zeros_like(r), torch.zeros_like(r[0])
    inside = torch.ones_like(r)
    for t in range(r.shape[0] - 1, -1, -1):
        go = 1.0 if s["done"] is None else 1.0 - s["done"][t].double()
        run_ = r[t] + GAMMA * go * v[t + 1] - v[t] + GAMMA * LAMBDA * go * run_
        if s["len"] is not None:
            inside[t] = (s["len"] > t).double().unsqueeze(1)
            run_ = run_ * inside[t]
        adv[t], ret[t] = run_, (run_ + v[t]) * inside[t]
    if not s["moments"]:
        return adv, ret
    k = inside.sum().clamp_min(1.0)
    mean = (adv * inside).sum() / k
    return adv, ret, torch.stack([mean, 1.0 / ((((adv - mean) * inside) ** 2).sum() / k).sqrt().add(1e-8)])


def _exact_act(s):
    sd = torch.exp(s["log_std"].double())
    z = s["noise"].double()
    # (the log-probability is that of the action as it is stored, in float32)
    act = s["mean"].double() + sd * z
    z = (act.float().double() - s["mean"].double()) / sd
    return act, -((z ** 2) / 2 + torch.log(sd * math.sqrt(2 * math.pi))).sum(-1)


def _exact_loss(s):
    """The loss in 64 bits, its gradients by differentiation."""
    mean, std = s["mean"].detach().double().requires_grad_(), s["log_std"].detach().double().requires_grad_()
    act = s["ring"].double().transpose(1, 2)
    sel = slice(None) if s["mask"] is None else s["mask"]
    with torch.enable_grad():
        dist = torch.exp(std).expand(mean.shape)
        lp = -(((act - mean) / dist) ** 2 / 2 + torch.log(dist) + math.log(2 * math.pi) / 2).sum(-1)[sel]
        old = s["log_pi_old"].double()[sel]
        ref = old if s["log_pi_ref"] is None else s["log_pi_ref"].double()[sel]
        adv = s["adv"].double()[sel]
        if s["moments"] is not None:
            adv = (adv - s["moments"][0].double()) * s["moments"][1].double()
        k = max(1, lp.numel())
        q = torch.exp(lp - old)
        inner = torch.where(adv >= 0, torch.clamp(q, max=1.0 + CLIP), torch.clamp(q, min=1.0 - CLIP)) * adv
        gain, kl = inner.sum() / k, (torch.exp(ref - lp) - 1.0 - (ref - lp)).sum() / k
        ent = (torch.log(dist) + (math.log(2 * math.pi) + 1.0) / 2).sum(-1)[sel].sum() / k
        loss = KL * kl - gain - ENTROPY * ent
    dmean, dstd = torch.autograd.grad(loss, (mean, std))
    cut = torch.where(adv > 0, q > 1.0 + CLIP, (q < 1.0 - CLIP) & (adv < 0)).double().sum() / k
    stats = torch.stack([gain.detach(), kl.detach(), ent.detach(), cut, q.detach().sum() / k, torch.tensor(float(lp.numel()), device=DEV, dtype=torch.float64)])
    return loss.detach(), stats, dmean, dstd


def work(case):
    op = case["op"]
    size = {"float32": 4, "bfloat16": 2}.get(case.get("dtype"), 4)
    if op == "scan":
        T, B, D = case["T"], case["B"], case["D"]
        n = T * B * D
        arrays, state = (6, 2 + 2 * case["h0"]) if case["train"] else (3, 1 + case["h0"])
        return {"bytes": arrays * n * size + state * B * D * 4 + (T * B if case["resets"] else 0) + (4 * B if case["lengths"] else 0),
                "flops": n * (24 if case["train"] else 9)}
    if op == "step":
        n = case["B"] * case["D"]
        return {"bytes": n * (3 * size + 8) + (case["B"] if case["resets"] else 0), "flops": 9 * n}
    if op == "advantages":
        n = case["T"] * case["E"] * case["n"]
        return {"bytes": 16 * n + 4 * case["E"] * case["n"] + (n if case["dones"] else 0) + (4 * case["E"] if case["lengths"] else 0), "flops": 8 * n}
    rows, A = case["B"] * case["n"], case["A"]
    std = A * size if case["shared_std"] else rows * A * size
    if op == "act":
        return {"bytes": rows * (A * (size + 8) + 4) + std, "flops": rows * A * 10}
    per = A * (2 * size + 4) + 8 + (4 if case["ref"] else 0) + (1 if case["mask"] else 0)
    return {"bytes": rows * per + 2 * std, "flops": rows * (A * 16 + 40)}
