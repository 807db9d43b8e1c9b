"""The clipped policy loss far from the recorded policy: ratios and KL terms over the range of double, with and without a KL
coefficient, against the same formulas in 64 bits, gradients by hand.

Bounds.  A row is computed in double and rounded once where it is stored: half a step of the result's type, 2^-24 or 2^-8, and
below the normal range half the smallest step.  In front of that: d = log_pi - log_pi_old to 2^-52 of its terms, some 600, so e^d
to 3e-13, and e^D - 1 and e^D - 1 - D lose at most a factor 50 of the last place more: 1e-12 of the sum of what is added, absolutely."""
import math

import pytest

import seq_oracle as so

pytestmark = pytest.mark.gpu


def _oracle(torch, mean, std, act, old, adv, ref, mask, clip, kl, ent):
    d_ = lambda t: t.detach().cpu().double()  # noqa: E731
    m, s, u = d_(mean), d_(std).expand(mean.shape), d_(act)
    z = (u - m) * torch.exp(-s)
    lp = (-z * z / 2 - s - math.log(2 * math.pi) / 2).sum(-1)
    d, A = lp - d_(old), d_(adv)
    D = (d_(old) if ref is None else d_(ref)) - lp
    q, em = torch.exp(d), torch.expm1(D)
    ok = torch.ones(lp.shape, dtype=torch.bool) if mask is None else mask.cpu()
    n = max(1, int(ok.sum()))
    cut = ((A > 0) & (q > 1 + clip)) | ((A < 0) & (q < 1 - clip))
    gain = torch.where(cut, q.clamp(1 - clip, 1 + clip) * A, q * A)
    k3 = em - D
    H = (s + (1 + math.log(2 * math.pi)) / 2).sum(-1)
    zero = torch.zeros((), dtype=torch.float64)
    mid = lambda t: torch.where(ok, t, zero).sum() / n  # noqa: E731
    rel = 1e-12
    klm, kla = (kl * mid(k3), kl * mid(k3.abs())) if kl else (zero, zero)
    loss = (-mid(gain) + klm - ent * mid(H), 1e-12 * (mid(gain.abs()) + ent * mid(H.abs())) + rel * kla)
    gq = torch.where(cut, zero, -q * A)
    g = torch.where(ok, (gq - (kl * em if kl else 0.0)) / n, zero).unsqueeze(-1)
    ga = torch.where(ok, (gq.abs() + (kl * em.abs() if kl else 0.0)) / n, zero).unsqueeze(-1)
    dm = (g * z * torch.exp(-s), rel * ga * (z * torch.exp(-s)).abs())
    w = torch.where(ok, 1.0 / n, zero).unsqueeze(-1)
    ds = (g * (z * z - 1) - ent * w, rel * (ga * (z * z + 1) + ent * w))
    if std.shape != mean.shape:
        ds = tuple(t.reshape(-1, mean.shape[-1]).sum(0) for t in ds)
    stats = (mid(gain), mid(k3), mid(H), mid(cut.double()), mid(q), ok.double().sum())
    return loss, dm, ds, stats


def _same(torch, got, want, extra, dtype, what):
    """Equal to half a step of the type; infinite where the value is beyond it."""
    got, big = got.detach().cpu().double(), want.to(dtype).double()
    inf = torch.isinf(big)
    assert torch.equal(got[inf], big[inf]), f"{what}: {got[inf][:4]} for {big[inf][:4]}"
    tol = extra + so.HALF[dtype] * (want.abs() + extra) + 2.0 ** -133 + 2.0 ** -150         # (2^-133: half of bfloat16's smallest step)
    so.within(got[~inf], want[~inf], tol[~inf], what)


CASES = [(d, s) for d in (-600.0, -300.0, -100.0, -89.0, -88.0, -20.0, 20.0, 88.0, 100.0) for s in (-1.0, 1.0)]


@pytest.mark.parametrize("kl", [0.0, 0.05, 1e-9])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("own_ref", [False, True])
@pytest.mark.parametrize("A,N", [(1, 40), (2, 40), (3, 900), (2, 9000), (7, 3000)])
def test_rows_far_from_the_recorded_policy(torch_cuda, A, N, own_ref, shared, kl):
    """One row in ordinary company, as far off as d says, in either advantage: finite losses and gradients where the formula's are."""
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    g = torch.Generator(device="cuda").manual_seed(A + N)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    for dtype in (torch.float32, torch.bfloat16):
        mean = (0.5 * rn(N, A)).to(dtype)
        std = ((rn(A) if shared else rn(N, A)) * 0.1 - 0.5).to(dtype)
        act = mean.float() + std.float().exp() * rn(N, A)
        lp = so.log_pi(mean, std, act).float().cuda()
        adv, mask = rn(N), torch.rand(N, device="cuda", generator=g) < 0.8
        for d, sign in CASES:
            old = lp + 0.2 * rn(N)
            ref = lp + 0.2 * rn(N) if own_ref else None
            k = N // 2
            a2, adv2 = act.clone(), adv.clone()
            mask[k] = True
            if d < 0:                                                   # an action that the policy of now finds very unlikely
                a2[k, 0] = mean[k, 0].float() + math.sqrt(-2 * d) * std.expand(N, A)[k, 0].float().exp()
            else:                                                       # or the recorded one did
                old[k] = lp[k] - d
            if own_ref:
                ref[k] = lp[k] + 0.1
            adv2[k] = sign
            m, s = mean.detach().requires_grad_(), std.detach().requires_grad_()
            loss, stats = clipped_policy_loss(m, s, a2, old, adv2, log_pi_ref=ref, mask=mask, kl_coef=kl, entropy_coef=0.01)
            dm, ds = torch.autograd.grad(loss, (m, s))
            wl, wm, ws, wst = _oracle(torch, mean, std, a2, old, adv2, ref, mask, 0.2, kl, 0.01)
            what = f"A={A} N={N} {dtype} d={d} adv={sign} kl={kl}"
            _same(torch, loss, *wl, torch.float32, what + " loss")
            _same(torch, dm, *wm, dtype, what + " dmean")
            _same(torch, ds, *ws, dtype, what + " dlog_std")
            for j, v in enumerate(wst):
                _same(torch, stats[j], v, 1e-12 * (v.abs() + 1 + A), torch.float32, f"{what} stats {j}")


def test_a_cut_row_has_no_gradient_however_far_off(torch_cuda):
    """e^D is beyond the range of float32 and the row is cut off: without a KL term it counts with its clipped gain alone."""
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    mean, std = torch.zeros(1, 1, device="cuda", requires_grad=True), torch.zeros(1, device="cuda", requires_grad=True)
    act, old, adv = torch.full((1, 1), 14.0, device="cuda"), torch.full((1,), -0.9, device="cuda"), torch.full((1,), -1.0, device="cuda")
    loss, stats = clipped_policy_loss(mean, std, act, old, adv)
    loss.backward()
    assert float(loss.detach()) == pytest.approx(0.8, abs=1e-7) and float(mean.grad) == 0.0 and float(std.grad) == 0.0
    assert float(stats[3]) == 1.0


def test_precision_of_whole_episodes(torch_cuda):
    """The loss and a shared deviation's gradient over many rows: rounded once, from sums in double."""
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    g = torch.Generator(device="cuda").manual_seed(2)
    N = 300000
    mean = torch.tanh(torch.randn(N, 2, device="cuda", generator=g))
    std = torch.tensor([-0.7, -0.5], device="cuda")
    act = mean + 0.1 * torch.randn(N, 2, device="cuda", generator=g) + std.exp() * torch.randn(N, 2, device="cuda", generator=g)
    old = so.log_pi(mean, std, act).float().cuda() + 0.2 * torch.randn(N, device="cuda", generator=g)
    adv = torch.randn(N, device="cuda", generator=g)
    m, s = mean.detach().requires_grad_(), std.detach().requires_grad_()
    loss, stats = clipped_policy_loss(m, s, act, old, adv, kl_coef=0.05, entropy_coef=0.01)
    dm, ds = torch.autograd.grad(loss, (m, s))
    wl, wm, ws, _ = _oracle(torch, mean, std, act, old, adv, None, None, 0.2, 0.05, 0.01)
    _same(torch, loss, *wl, torch.float32, "loss")
    _same(torch, dm, *wm, torch.float32, "dmean")
    _same(torch, ds, *ws, torch.float32, "dlog_std")


def test_a_reference_that_begins_where_the_old_policy_does(torch_cuda):
    """Two views of one buffer that begin at the same element are still two tensors."""
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    for lead in ((50,), (6000,), (40, 30)):
        N = math.prod(lead)
        mean, std = torch.zeros(*lead, 1, device="cuda"), torch.zeros(1, device="cuda")
        act, adv = torch.randn(*lead, 1, device="cuda"), torch.randn(lead, device="cuda")
        rows = so.log_pi(mean, std, act).float().cuda() + 0.2 * torch.randn(lead, device="cuda")
        rows.view(-1)[0] = -1.0
        one = rows.view(-1)[:1].expand(N).view(lead) if len(lead) == 1 else rows[:1, :1].expand(lead)
        for old, ref in ((one, rows), (rows, one)):
            got = clipped_policy_loss(mean, std, act, old, adv, log_pi_ref=ref, kl_coef=0.3)
            want = clipped_policy_loss(mean, std, act, old.clone(), adv, log_pi_ref=ref.clone(), kl_coef=0.3)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), lead


def test_more_gradient_values_than_2_to_the_29(torch_cuda):
    """2^28 + 1 rows of two components, all alike (expanded inputs): their gradients, scaled by an upstream gradient of a half."""
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    N = (1 << 28) + 1
    m = torch.tensor([[0.1, -0.2]], device="cuda").expand(N, 2).detach().requires_grad_()
    s = torch.tensor([-0.5, -0.4], device="cuda").requires_grad_()
    act, one = torch.tensor([[0.3, 0.1]], device="cuda").expand(N, 2), torch.ones(1, device="cuda").expand(N)
    loss, _ = clipped_policy_loss(m, s, act, -1.5 * one, -one)
    dm, ds = torch.autograd.grad(loss, (m, s), torch.tensor(0.5, device="cuda"))
    z = (act[0].cpu().double() - m[0].detach().cpu().double()) * torch.exp(-s.detach().cpu().double())
    q = torch.exp((-z * z / 2 - s.detach().cpu().double() - math.log(2 * math.pi) / 2).sum() + 1.5)
    want = 0.5 * q / N * z * torch.exp(-s.detach().cpu().double())      # (q is not clipped: the advantage is negative and q above 1)
    assert float(q) > 1.0
    so.within(dm[0], want, 2 * so.U * want.abs(), "dmean")              # two roundings: stored, scaled
    assert bool((dm == dm[0]).all())
    so.within(ds, 0.5 * q * (z * z - 1), 2 * so.U * (q * (z * z - 1)).abs() + 1e-9, "dlog_std")
