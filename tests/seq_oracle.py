"""Plain 64-bit forms of the sequence operators (marl_amd.recurrence, marl_amd.policy_loss) with error bounds, for their
tests: step by step on the CPU, in float64, written from the formulas.

Bounds.  u = 2^-24 is half a step of float32.  Everything the float32 kernels do is a chain of maps y = A y + S whose terms
are bounded by the same chain on absolute values, Y = A Y + |S| (sums may cancel, the bound does not); a step adds at most
C u Y to the error and passes A times the error it got.  C = 16 covers a step's roundings: the exponential (at most 2 steps),
1 + e, the reciprocal, the product (together at most 5 u on a and on 1 - a, which enter A, S and, once more, the composition of
stretches), the product (1 - a) x, the multiply-add, and the same three again when a stretch is walked a second time."""
import math

import torch

U = 2.0 ** -24
C = 16.0
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _tb(t, batch_first):
    return t.detach().cpu().double().transpose(0, 1) if batch_first else t.detach().cpu().double()


def scan(gate, x, h0=None, resets=None, lengths=None, batch_first=False, dh=None, dlast=None):
    """Values and elementwise bounds: dict of name -> (value, bound), laid out as the operator's outputs."""
    dt = gate.dtype
    g, xx = _tb(gate, batch_first), _tb(x, batch_first)
    T, B, D = g.shape
    n = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    cut = torch.zeros(T, B, dtype=torch.bool) if resets is None else (_tb(resets, batch_first) != 0)
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.detach().cpu().double()
    H, e = h.abs(), torch.zeros_like(h)
    outs, tols, prev, prevH, preve = [], [], [], [], []
    a, b = torch.sigmoid(g), torch.sigmoid(-g)
    zero = torch.zeros((), dtype=torch.float64)
    for t in range(T):
        c = cut[t].unsqueeze(1)
        k, kH, ke = torch.where(c, zero, h), torch.where(c, zero, H), torch.where(c, zero, e)
        prev.append(k); prevH.append(kH); preve.append(ke)
        nh = a[t] * k + b[t] * xx[t]
        nH = a[t] * kH + b[t] * xx[t].abs()
        ne = a[t] * ke + C * U * nH
        on = (t < n).unsqueeze(1)
        outs.append(torch.where(on, nh, zero)); tols.append(torch.where(on, ne + HALF[dt] * nh.abs() * (dt != torch.float32), zero))
        h, H, e = torch.where(on, nh, h), torch.where(on, nH, H), torch.where(on, ne, e)
    first = lambda s: (torch.stack(s) if s else torch.zeros(T, B, D, dtype=torch.float64)).transpose(0, 1) if batch_first else (torch.stack(s) if s else torch.zeros(T, B, D, dtype=torch.float64))  # noqa: E731
    res = {"h": (first(outs), first(tols)), "last": (h, e)}
    if dh is None and dlast is None:
        return res
    d = torch.zeros(T, B, D, dtype=torch.float64) if dh is None else _tb(dh, batch_first)
    cg = torch.zeros(B, D, dtype=torch.float64) if dlast is None else dlast.cpu().double()
    cG, ce = cg.abs(), torch.zeros_like(cg)
    dg, dx, tg, tx = ([None] * T for _ in range(4))
    for t in range(T - 1, -1, -1):
        on, c = (t < n).unsqueeze(1), cut[t].unsqueeze(1)
        G, GG, Ge = d[t] + cg, d[t].abs() + cG, ce + U * (d[t].abs() + cG)
        w = a[t] * b[t]
        stored = preve[t] + (HALF[dt] * prev[t].abs() if dt != torch.float32 and t > 0 else 0.0)       # (h is kept in the outputs' type)
        m, mm = prev[t] - xx[t], prevH[t] + xx[t].abs()
        vx, vg = G * b[t], G * m * w
        ex = Ge * b[t] + C * U * GG * b[t]
        eg = Ge * m.abs() * w + GG * w * (stored + C * U * mm)
        r = HALF[dt] if dt != torch.float32 else 0.0
        dx[t], tx[t] = torch.where(on, vx, zero), torch.where(on, ex + r * (vx.abs() + ex), zero)
        dg[t], tg[t] = torch.where(on, vg, zero), torch.where(on, eg + r * (vg.abs() + eg), zero)
        nG, nGG, nGe = a[t] * G, a[t] * GG, a[t] * Ge + C * U * a[t] * GG
        nG, nGG, nGe = (torch.where(c, zero, v) for v in (nG, nGG, nGe))
        cg, cG, ce = torch.where(on, nG, cg), torch.where(on, nGG, cG), torch.where(on, nGe, ce)
    res.update(dgate=(first(dg), first(tg)), dx=(first(dx), first(tx)), dh0=(cg, ce))
    return res


def advantages(rewards, values, dones=None, lengths=None, gamma=0.95, lam=0.95):
    r, v = rewards.cpu().double(), values.cpu().double()
    gamma, lam = float(torch.tensor(gamma, dtype=torch.float32)), float(torch.tensor(lam, dtype=torch.float32))     # as the entry point takes them
    T, E = r.shape[:2]
    n = torch.full((E,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    n = n.view(E, *([1] * (r.dim() - 2)))
    zero = torch.zeros((), dtype=torch.float64)
    adv, ret, ta = torch.zeros_like(r), torch.zeros_like(r), torch.zeros_like(r)
    y, Y, e = torch.zeros_like(r[0]), torch.zeros_like(r[0]), torch.zeros_like(r[0])
    for t in range(T - 1, -1, -1):
        done = torch.zeros_like(r[0], dtype=torch.bool) if dones is None else dones[t].cpu() != 0
        nv = torch.where(done, zero, v[t + 1])
        ny = r[t] + gamma * nv - v[t] + gamma * lam * torch.where(done, zero, y)
        nY = r[t].abs() + gamma * nv.abs() + v[t].abs() + gamma * lam * torch.where(done, zero, Y)
        ne = gamma * lam * torch.where(done, zero, e) + C * U * nY
        on = (t < n).expand_as(y)
        y, Y, e = torch.where(on, ny, zero), torch.where(on, nY, zero), torch.where(on, ne, zero)
        adv[t], ta[t], ret[t] = y, e, torch.where(on, y + v[t], zero)
    inside = (torch.arange(T).view(T, *([1] * (r.dim() - 1))) < n.unsqueeze(0)).expand_as(r)
    x = adv[inside]
    mean = x.mean() if x.numel() else zero
    sd = ((x - mean) ** 2).mean().sqrt() if x.numel() else zero
    ret_tol = torch.where(inside, ta + U * (ret.abs() + ta), zero)
    return adv, ta, ret, ret_tol, mean, sd


def policy_loss(mean, log_std, actions, old, adv, ref=None, mask=None, moments=None, clip=0.2, kl=0.0, ent=0.0):
    """loss, stats, gradients by differentiation, all in float64, and the sum of the terms' magnitudes."""
    d = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    m, s = d(mean).requires_grad_(), d(log_std).requires_grad_()
    rows = torch.ones(m.shape[:-1], dtype=torch.bool) if mask is None else mask.cpu() != 0
    sf = s.expand(m.shape)[rows]
    z = (d(actions)[rows] - m[rows]) / torch.exp(sf)
    lp = (-z * z / 2 - sf - math.log(2 * math.pi) / 2).sum(-1)
    o = d(old)[rows]
    a = d(adv)[rows]
    if moments is not None:
        mo = d(moments)
        a = (a - mo[0]) * mo[1]
    D = (o if ref is None else d(ref)[rows]) - lp
    q = torch.exp(lp - o)
    gain = torch.minimum(q * a, q.clamp(1 - clip, 1 + clip) * a)
    k3 = torch.expm1(D) - D
    H = (sf + (1 + math.log(2 * math.pi)) / 2).sum(-1)
    n = max(1, int(rows.sum()))
    loss = (-gain + kl * k3 - ent * H).sum() / n
    cut = ((a > 0) & (q > 1 + clip)) | ((a < 0) & (q < 1 - clip))
    if int(rows.sum()):
        dm, ds = torch.autograd.grad(loss, (m, s), allow_unused=True)
        ds = torch.zeros_like(s) if ds is None else ds
    else:
        dm, ds = torch.zeros_like(m), torch.zeros_like(s)
    stats = torch.stack([gain.sum() / n, k3.sum() / n, H.sum() / n, cut.double().sum() / n, q.sum() / n, rows.sum().double()]).detach()
    size = ((q * a).abs() + kl * k3.abs() + ent * H.abs()).sum() / n
    return loss.detach(), stats, dm, ds, float(size.detach())


def log_pi(mean, log_std, actions):
    m, s, a = mean.detach().cpu().double(), log_std.detach().cpu().double(), actions.cpu().double()
    z = (a - m) / torch.exp(s)
    return (-z * z / 2 - s - math.log(2 * math.pi) / 2).sum(-1)


def within(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, wanted {tuple(want.shape)}"
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off / torch.as_tensor(tol).clamp_min(1e-300)).nan_to_num(posinf=1e9).max()):.3g} times the bound"
