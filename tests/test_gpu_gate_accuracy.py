"""How exact the gate's two weights are, a = sigmoid(g) and b = 1 - a, over the whole range of g.

With u = 2^-24 and t = e^-|g|: |g| log2(e) minus a whole number is kept to 2^-24 (two fused products, each rounded below 1), that is
0.7 u of t; the hardware's exponential is good to one unit in the last place, 2 u.  1 + t: u and at most half of t's 2.7 u.  A
reciprocal with a Newton step: u.  So the larger weight, 1 / (1 + t), is good to 3.4 u; the smaller, t / (1 + t), to 2.7 u for t
and u each for the sum, the reciprocal and the product: 5.7 u.  Held to 6 u, and one step of the smallest numbers, 2^-149."""
import pytest

import seq_oracle as so

pytestmark = pytest.mark.gpu


def test_weights_over_the_whole_range(torch_cuda):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan, gated_scan_step
    g = torch.cat((torch.linspace(-110, 110, 65536 - 6), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-5, -1e-5]))).cuda().view(256, 256)
    one, zero = torch.ones_like(g), torch.zeros_like(g)
    a, b = torch.sigmoid(g.cpu().double()), torch.sigmoid(-g.cpu().double())
    tiny = 2.0 ** -149
    so.within(gated_scan_step(g, zero, one.clone()), a, 6 * so.U * a + tiny, "a, step")
    so.within(gated_scan_step(g, one, zero.clone()), b, 6 * so.U * b + tiny, "1 - a, step")
    so.within(gated_scan(g.unsqueeze(0), zero.unsqueeze(0), one)[0][0], a, 6 * so.U * a + tiny, "a, scan")
    so.within(gated_scan(g.unsqueeze(0), one.unsqueeze(0))[0][0], b, 6 * so.U * b + tiny, "1 - a, scan")


def test_gates_that_are_no_numbers(torch_cuda):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan_step
    nan = float("nan")
    g = torch.tensor([[nan, -nan, 1e38, -1e38]], device="cuda")
    out = gated_scan_step(g, torch.full_like(g, 3.0), torch.full_like(g, 7.0))[0].tolist()
    assert out[0] != out[0] and out[1] != out[1] and out[2:] == [7.0, 3.0]
