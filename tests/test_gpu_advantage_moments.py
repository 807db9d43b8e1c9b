"""The moments of advantages far from zero: against two passes in 64 bits over the very advantages that were returned, so that only
the moments' own arithmetic shows.  Double throughout: d^2 terms and means to 1e-13 of themselves, the deviation so, and one rounding to
float32 of each result; a deviation of d takes the rounding of the mean it is measured from, 2^-52 of the mean, at most."""
import pytest

import seq_oracle as so

pytestmark = pytest.mark.gpu


def _check(torch, adv, mom, inside, what):
    x = adv.cpu().double()[inside.cpu()]
    mean = x.mean()
    sd = ((x - mean) ** 2).mean().sqrt()
    want = 1.0 / (sd + 1e-8)
    assert abs(float(mom[0]) - float(mean)) <= (so.U + 1e-12) * abs(float(mean)), what
    # an error e of the deviation moves 1 / (sd + 1e-8) by e times its square
    e = 1e-12 * float(sd) + 2.0 ** -50 * abs(float(mean))
    assert abs(float(mom[1]) - float(want)) <= (so.U + 1e-12) * float(want) + 1.01 * e * float(want) ** 2, (what, float(mom[1]), float(want))


@pytest.mark.parametrize("T,E,n", [(1, 1, 1), (1, 64, 30), (200, 3, 5), (40, 2300, 30), (1000, 2, 7), (7, 1, 1)])
def test_advantages_far_from_zero(torch_cuda, T, E, n):
    torch = torch_cuda
    from marl_amd.recurrence import advantages
    g = torch.Generator(device="cuda").manual_seed(T + E)
    for offset, noise in ((0.0, 1.0), (100.0, 0.01), (12345.678, 0.01), (0.3, 0.0), (777.7, 0.0)):
        r = offset + noise * torch.randn(T, E, n, device="cuda", generator=g)
        v = torch.zeros(T + 1, E, n, device="cuda")                     # (gamma 0: the advantage is the reward)
        lengths = torch.randint(0, T + 1, (E,), device="cuda", generator=g, dtype=torch.int32)
        for le in (None, lengths):
            adv, _, mom = advantages(r, v, lengths=le, gamma=0.0, lam=0.5, moments=True)
            inside = torch.ones(T, E, n, dtype=torch.bool, device="cuda") if le is None else (torch.arange(T, device="cuda").view(T, 1, 1) < le.view(1, E, 1)).expand(T, E, n)
            if not bool(inside.any()):
                assert mom.tolist() == [0.0, pytest.approx(1e8)]
                continue
            _check(torch, adv, mom, inside, (offset, noise, le is None))
            again = advantages(r, v, lengths=le, gamma=0.0, lam=0.5, moments=True)[2]
            assert torch.equal(mom, again)


def test_one_value_that_is_no_number_shows(torch_cuda):
    torch = torch_cuda
    from marl_amd.recurrence import advantages
    r, v = torch.randn(50, 4, 3, device="cuda"), torch.zeros(51, 4, 3, device="cuda")
    r[20, 1, 1] = float("nan")
    mom = advantages(r, v, gamma=0.0, moments=True)[2]
    assert bool(torch.isnan(mom).all())
