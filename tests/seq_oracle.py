"""Plain 64-bit forms of the sequence operators (marl_amd.recurrence, marl_amd.policy_loss) with error bounds, for their
tests: step by step on the CPU, in float64, written from the formulas.

Bounds.  u = 2^-24 is half a step of float32.  Everything the float32 kernels do is a chain of maps y = A y + S whose terms
are bounded by the same chain on absolute values, Y = A Y + |S| (sums may cancel, the bound does not); a step adds at most
C u Y to the error and passes A times the error it got.  What a step rounds: exp(-g) is 2^t with t = g log2(e) rounded (and that
constant itself): 1.25 |g| of u on e, and 2 for the hardware's exponential; 1 + e, the reciprocal (2), the product or the
difference: together at most 6 + 1.25 |g| on a and on 1 - a; the product (1 - a) x and the multiply-add 2 more.  The
composition of stretches walks a step a second time: twice that, C = 16 + 2.5 |g|; where |g| > 40, e is below u or above 1 / u and its own
error no longer shows (a or 1 - a rounds to 1) except in the smaller of the two, whose terms are below u Y."""
import math

import torch

U = 2.0 ** -24
def C(g):
    return 16.0 + 2.5 * g.abs().clamp(max=40.0)


CA = 16.0                                                               # the advantages have no gate
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
        ne = a[t] * ke + C(g[t]) * U * nH
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
        ex = Ge * b[t] + C(g[t]) * U * GG * b[t]
        eg = Ge * m.abs() * w + GG * w * (stored + 2 * C(g[t]) * U * mm)
        r = HALF[dt] if dt != torch.float32 else 0.0
        dx[t], tx[t] = torch.where(on, vx, zero), torch.where(on, ex + r * (vx.abs() + ex), zero)
        dg[t], tg[t] = torch.where(on, vg, zero), torch.where(on, eg + r * (vg.abs() + eg), zero)
        nG, nGG, nGe = a[t] * G, a[t] * GG, a[t] * Ge + C(g[t]) * U * a[t] * GG
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
        ne = gamma * lam * torch.where(done, zero, e) + CA * U * nY
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
    """(value, bound) of loss, stats and the gradients (by differentiation), in float64.

    Bounds.  log_pi, d and the clipping decision are in double in the kernel; from there on a row is float32.  Per row, in units
    of u: q = e^d: |d| for d's rounding, 3 for the exponential; A = (adv - mean) / deviation: 2; so a factor of 10 + |d| covers
    q A, the clipped one and the products with them.  e^D - 1: |D| (1 + e^D) for D's rounding and the last place of its terms,
    a factor of 16 with its own; e^D - 1 - D: 16 of itself below |D| = 1 (its series is a product of D with at most ten
    roundings), and of e^D + 1 + |D| beyond.  Products with z and e^-s: 4 more.  Sums are in double."""
    d_ = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    m, s = d_(mean).requires_grad_(), d_(log_std).requires_grad_()
    rows = torch.ones(m.shape[:-1], dtype=torch.bool) if mask is None else mask.cpu() != 0
    sf = s.expand(m.shape)[rows]
    z = (d_(actions)[rows] - m[rows]) / torch.exp(sf)
    lp = (-z * z / 2 - sf - math.log(2 * math.pi) / 2).sum(-1)
    o = d_(old)[rows]
    a = d_(adv)[rows]
    if moments is not None:
        mo = d_(moments)
        a = (a - mo[0]) * mo[1]
    D = (o if ref is None else d_(ref)[rows]) - lp
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
    with torch.no_grad():
        d, e, w = lp - o, torch.exp(D), 1.0 / n
        e_gain = U * (q * a).abs() * (10 + d.abs())
        e_k3 = 16 * U * torch.where(D.abs() < 1, k3, e + 1 + D.abs() * (1 + e))
        e_g = w * (torch.where(cut, torch.zeros_like(e_gain), e_gain) + kl * 16 * U * (torch.expm1(D).abs() + D.abs() * (1 + e)))
        g = w * (torch.where(cut, torch.zeros_like(q), -q * a) - kl * torch.expm1(D))
        r_m = (e_g + 4 * U * g.abs()).unsqueeze(-1) * (z / torch.exp(sf)).abs()
        r_s = (e_g + 4 * U * g.abs()).unsqueeze(-1) * (z * z + 1) + 3 * U * ent * w
        b_m, b_s = torch.zeros_like(m), torch.zeros(m.shape, dtype=torch.float64)
        b_m[rows], b_s[rows] = r_m, r_s
        if s.shape != m.shape:
            b_s = b_s.reshape(-1, m.shape[-1]).sum(0)
        stats = torch.stack([gain.sum() / n, k3.sum() / n, H.sum() / n, cut.double().sum() / n, q.sum() / n, rows.sum().double()])
        b_stats = torch.stack([e_gain.sum() / n, e_k3.sum() / n, 0 * H.sum(), 0 * H.sum(), (U * q * (4 + d.abs())).sum() / n, 0 * H.sum()])
        b_loss = b_stats[0] + kl * b_stats[1]
        tiny = 1e-13 * (H.abs().sum() / n + 1)                           # the sums themselves
    return ((loss.detach(), b_loss + U * loss.detach().abs() + tiny), (stats, b_stats + U * stats.abs() + tiny),
            (dm, b_m), (ds, b_s + 1e-13 * b_s / U))


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
