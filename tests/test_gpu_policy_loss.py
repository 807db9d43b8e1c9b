"""The clipped policy loss and the sampling of actions (marl_amd.policy_loss) against their 64-bit forms.

Bounds: seq_oracle.policy_loss's for the float32 arithmetic of a row, and the rounding of each result: half a step of its type,
2^-24 for float32; a bfloat16 gradient is rounded from float32, 2^-8.  An upstream gradient other than 1 multiplies the
stored one: once more the same."""
import gc
import math

import pytest

import seq_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_garbage():
    """A HIP graph that the garbage collector frees while another one is captured ends the process (its destructor may not
    run then): none is left from tests before, and none to tests after."""
    gc.collect()
    yield
    gc.collect()


U = so.U


def _make(torch, lead, A, dtype, shared, seed, ref=False, mask=None, spread=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    dt = getattr(torch, dtype)
    mean = torch.tanh(rn(*lead, A)).to(dt)
    std = ((rn(A) if shared else rn(*lead, A)) * 0.3 - 0.6).to(dt)
    act = mean.float() + 0.1 * rn(*lead, A) + std.float().exp() * rn(*lead, A)
    lp = so.log_pi(mean, std, act).float().cuda()
    old = lp + spread * rn(*lead)
    rf = lp + spread * rn(*lead) if ref else None
    adv = 2 * rn(*lead) + 0.3
    mk = None if mask is None else torch.rand(*lead, device="cuda", generator=g) < mask
    return mean, std, act, old, adv, rf, mk


def _check(torch, mean, std, act, old, adv, ref, mask, moments=None, clip=0.2, kl=0.1, ent=0.02, up=None, what=""):
    from marl_amd.policy_loss import clipped_policy_loss
    m, s = mean.detach().requires_grad_(), std.detach().requires_grad_()
    loss, stats = clipped_policy_loss(m, s, act, old, adv, log_pi_ref=ref, mask=mask, adv_moments=moments, clip=clip, kl_coef=kl, entropy_coef=ent)
    dm, ds = torch.autograd.grad(loss if up is None else loss * up, (m, s))
    wl, wst, wm, ws = so.policy_loss(mean, std, act, old, adv, ref, mask, moments, clip, kl, ent)
    so.within(loss, *wl, f"{what} loss")
    so.within(stats, *wst, f"{what} stats")
    half, f = so.HALF[mean.dtype], 1.0
    if up is not None:
        f = float(torch.tensor(up, dtype=torch.float32))
    tiny = 1.2e-38                                                       # results below the normal range of float32 and bfloat16
    for got, (want, bound), name in ((dm, wm, "dmean"), (ds, ws, "dlog_std")):
        t = bound + half * (want.abs() + bound)
        if up is not None:
            t = t + half * (want.abs() + t)
        so.within(got, want * f, abs(f) * t + tiny, f"{what} {name}")
    return loss, stats, dm, ds


LEADS = [(1,), (63,), (5, 7), (2048,), (4096,), (4097,), (3, 5, 30), (17, 40, 30), (300, 64)]


@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lead", LEADS)
def test_loss_matches_the_64_bit_form(torch_cuda, lead, dtype, shared):
    torch = torch_cuda
    for A in (1, 2, 3, 4, 5, 8, 13, 32) if math.prod(lead) < 5000 else (2, 3, 7, 32):
        for ref, mask in ((False, None), (True, 0.7)):
            c = _make(torch, lead, A, dtype, shared, A + len(lead), ref, mask)
            mom = torch.tensor([0.3, 0.45], device="cuda") if ref else None
            _check(torch, *c, moments=mom, what=f"{lead} A={A} ref={ref}")


def test_loss_of_replay_views(torch_cuda):
    """Actions as a ring keeps them (T, E, A, n), masks and advantages cut out of larger tensors, expanded inputs."""
    torch = torch_cuda
    T, E, n, A = 12, 20, 30, 2
    mean, std, act, old, adv, ref, mask = _make(torch, (T, E, n), A, "float32", True, 9, True, 0.8)
    ring = act.transpose(-1, -2).contiguous()
    wide = torch.zeros(T, E, 2, n, device="cuda")
    wide[:, :, 1] = adv
    a = _check(torch, mean, std, ring.transpose(-1, -2), old, wide[:, :, 1], ref, mask, what="ring")
    b = _check(torch, mean, std, act, old, adv, ref, mask, what="rows")
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    tl = torch.randn(E, T, n, device="cuda").transpose(0, 1)            # cannot be walked with one stride: copied
    _check(torch, mean, std, act, old, tl, ref, mask.transpose(0, 1).contiguous().transpose(0, 1), what="swapped axes")
    one = torch.full((1, 1, 1), 0.7, device="cuda").expand(T, E, n)
    _check(torch, mean, std, act, old, one, old, None, what="expanded")
    m2 = torch.randn(T, E, n, 3 * A, device="cuda")[..., 1::3]
    _check(torch, m2, std, act, old, adv, None, None, what="strided mean")
    _check(torch, mean, std, act, old, adv, ref, mask, clip=1.5, what="clip beyond 1")
    _check(torch, mean[0, 0, 0], std, act[0, 0, 0], old[0, 0, 0], adv[0, 0, 0], ref[0, 0, 0], None, what="one row, no axes")
    both = torch.randn(T, E, n, 2 * A, device="cuda") * 0.3             # one head's output, cut in two
    _check(torch, both[..., :A], both[..., A:], act, old, adv, ref, mask, what="cut head")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_upstream_gradients_and_retained_graphs(torch_cuda, dtype):
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    for lead in ((50,), (6000,)):
        c = _make(torch, lead, 2, dtype, True, 4, True, 0.6)
        _check(torch, *c, up=-0.37, what="scaled")
        m, s = c[0].detach().requires_grad_(), c[1].detach().requires_grad_()
        loss, _ = clipped_policy_loss(m, s, *c[2:5], kl_coef=0.1)
        first = torch.autograd.grad(loss, (m, s), retain_graph=True)
        keep = [t.clone() for t in first]
        twice = torch.autograd.grad(loss * 2.0, (m, s), retain_graph=True)
        again = torch.autograd.grad(loss, (m, s))
        for f, k, t, a in zip(first, keep, twice, again):
            assert torch.equal(f, k) and torch.equal(f, a) and torch.equal(t, 2 * f)       # (times two is exact)


def test_no_valid_rows_and_values_that_do_not_count(torch_cuda):
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    for lead in ((40,), (7000,), (0,)):
        mean, std, act, old, adv, ref, _ = _make(torch, lead, 3, "float32", False, 2, True)
        none = torch.zeros(lead, dtype=torch.bool, device="cuda")
        m, s = mean.clone().requires_grad_(), std.clone().requires_grad_()
        loss, stats = clipped_policy_loss(m, s, act * float("nan"), old, adv, log_pi_ref=ref, mask=none, kl_coef=0.2, entropy_coef=0.1)
        loss.backward()
        assert float(loss.detach()) == 0.0 and not bool(stats.any()) and not bool(m.grad.any()) and not bool(s.grad.any())
        if not lead[0]:
            continue
        mask = torch.rand(lead, device="cuda") < 0.5
        want = _check(torch, mean, std, act, old, adv, ref, mask, what="clean")
        bad = [t.clone() for t in (mean, std, act, old, adv, ref)]
        for t, v in zip(bad, (float("nan"), float("inf"), float("inf"), -float("inf"), float("nan"), float("nan"))):
            t[~mask] = v
        m, s = bad[0].requires_grad_(), bad[1].requires_grad_()
        loss, stats = clipped_policy_loss(m, s, bad[2], bad[3], bad[4], log_pi_ref=bad[5], mask=mask, clip=0.2, kl_coef=0.1, entropy_coef=0.02)
        got = (loss, stats) + torch.autograd.grad(loss, (m, s))
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        # one NaN that does count shows
        adv2 = adv.clone(); adv2[mask.nonzero()[0]] = float("nan")
        assert math.isnan(float(clipped_policy_loss(mean, std, act, old, adv2, mask=mask)[0].detach()))


def test_ratios_at_the_clipping_border(torch_cuda):
    """Ratios within 1e-7 of the border on either side fall where the 64-bit form puts them."""
    torch = torch_cuda
    N = 6000
    g = torch.Generator(device="cuda").manual_seed(1)
    mean = torch.zeros(N, 1, device="cuda"); std = torch.zeros(1, device="cuda")
    act = torch.randn(N, 1, device="cuda", generator=g)
    lp = so.log_pi(mean, std, act)
    edge = torch.log(torch.where(torch.arange(N) % 2 == 0, 1.2, 0.8).double())
    old = (lp - edge + 1e-7 * torch.randn(N, dtype=torch.float64)).float().cuda()
    adv = torch.randn(N, device="cuda", generator=g)
    _check(torch, mean, std, act, old, adv, None, None, what="border")


def test_loss_gradients_against_differences(torch_cuda):
    torch = torch_cuda
    mean, std, act, old, adv, ref, mask = _make(torch, (12,), 2, "float32", False, 3, True, 0.8)
    _, _, dm, ds = _check(torch, mean, std, act, old, adv, ref, mask, what="formula")
    bounds = [w[1] for w in so.policy_loss(mean, std, act, old, adv, ref, mask, None, 0.2, 0.1, 0.02)[2:]]
    step = 1e-6
    for k, grad in ((0, dm), (1, ds)):
        for j in range(mean.numel()):
            vals = []
            for sgn in (1, -1):
                a = [mean.double(), std.double()]
                a[k] = a[k].clone()
                a[k].view(-1)[j] += sgn * step
                vals.append(float(so.policy_loss(a[0], a[1], act, old, adv, ref, mask, None, 0.2, 0.1, 0.02)[0][0]))
            d = (vals[0] - vals[1]) / (2 * step)
            # truncation step^2 times a third derivative below 1e3, cancellation 1e-16 x 10 / step, the kernel's own bound and one rounding
            assert abs(float(grad.view(-1)[j]) - d) <= 2e-9 + 1e-8 + float(bounds[k].view(-1)[j]) + U * abs(d), (k, j)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("E,n,A,shared", [(1, 1, 1, True), (5, 30, 2, True), (4096, 30, 2, True), (3, 1024, 7, False), (2, 13, 32, False)])
def test_actions_and_their_log_pi(torch_cuda, E, n, A, shared, dtype):
    torch = torch_cuda
    from marl_amd.policy_loss import gaussian_act, gaussian_log_pi
    mean, std, *_ = _make(torch, (E, n), A, dtype, shared, 5)
    noise = torch.randn(E, n, A, device="cuda")
    ring, lp = torch.full((2, E, A, n), 9.0, device="cuda"), torch.full((E, 1, n), 9.0, device="cuda")
    act, got = gaussian_act(mean, std, noise, actions=ring[1].transpose(-1, -2), log_pi=lp[:, 0])
    assert act.data_ptr() == ring[1].data_ptr() and bool((ring[0] == 9.0).all())
    sd = std.detach().cpu().double().exp()
    want = mean.cpu().double() + sd * noise.cpu().double()
    so.within(act, want, U * want.abs() + 1e-14 * (want.abs() + sd * noise.cpu().double().abs()), "actions")
    wl = so.log_pi(mean, std, act)
    so.within(got, wl, U * wl.abs() + 1e-11 * A, "log_pi")
    again = gaussian_log_pi(mean, std, act)
    assert torch.equal(again, got)                                      # a ratio against the stored value starts at 1
    plain, lp2 = gaussian_act(mean, std, noise)
    assert torch.equal(plain, act) and torch.equal(lp2, got)


def test_captured_graphs(torch_cuda, no_garbage):
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss, gaussian_act
    c = _make(torch, (50, 200), 2, "float32", True, 8, True, 0.5)       # (several workgroups, a mask: a workspace is in use)
    m, s = c[0].requires_grad_(), c[1].requires_grad_()
    up = torch.full((), 0.5, device="cuda")

    def work():
        loss, stats = clipped_policy_loss(m, s, *c[2:5], log_pi_ref=c[5], mask=c[6], kl_coef=0.1, entropy_coef=0.01)
        return (loss.detach(), stats) + torch.autograd.grad(loss, (m, s), up) + gaussian_act(m, s, c[2])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = work()
    for k in range(3):
        with torch.no_grad():
            m.copy_(torch.tanh(torch.randn_like(m)))
            c[4].copy_(torch.randn_like(c[4]))
            c[6].copy_(torch.rand_like(c[4]) < 0.3 * k)                 # the first replay: no valid row
            up.fill_(1.0 if k == 1 else 0.25)
        g.replay()
        eager = work()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k


def test_backward_notices_inputs_overwritten_since(torch_cuda):
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss, gaussian_act
    mean, std, act, old, adv, _, _ = _make(torch, (8,), 2, "float32", True, 6)
    m = mean.requires_grad_()
    loss, _ = clipped_policy_loss(m, std, act, old, adv)
    gaussian_act(m, std, torch.randn(8, 2, device="cuda"), log_pi=old)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
