"""The gated memory and the advantages (marl_amd.recurrence) against their 64-bit forms, elementwise, at bounds derived
there: lengths from none to many tiles, odd widths, strided and expanded tensors, resets, values that must not be read,
offsets beyond 32 bits, streams and HIP graphs."""
import gc

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


SHAPES = [(1, 1, 1), (0, 3, 5), (3, 2, 64), (31, 3, 7), (32, 1, 65), (33, 2, 12), (100, 5, 61), (200, 64, 30),
          (9, 300, 256), (67, 280, 256), (40, 1100, 61), (1000, 2, 5), (4099, 1, 3), (700, 3, 256),
          (1, 1200, 256), (8, 1200, 256), (21, 601, 256), (24, 1200, 256), (35, 1201, 256), (600, 1, 64), (90, 20, 64)]


def _make(torch, T, B, D, dtype, batch_first, seed, resets=False, lengths=False, h0=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    lead = (B, T) if batch_first else (T, B)
    gate, x = (2 * rn(*lead, D) + 1).to(dtype), (3 * rn(*lead, D)).to(dtype)
    r = torch.rand(*lead, device="cuda", generator=g) < 0.1 if resets else None
    n = torch.randint(0, T + 1, (B,), device="cuda", generator=g, dtype=torch.int32) if lengths else None
    return gate, x, (rn(B, D) if h0 else None), r, n


def _check(torch, gate, x, h0, r, n, bf, seed=0, what=""):
    from marl_amd.recurrence import gated_scan
    g = torch.Generator(device="cuda").manual_seed(seed + 77)
    leaves = [t.detach().requires_grad_() for t in (gate, x)] + ([] if h0 is None else [h0.detach().requires_grad_()])
    h, last = gated_scan(leaves[0], leaves[1], leaves[2] if h0 is not None else None, resets=r, lengths=n, batch_first=bf)
    dh = torch.randn(h.shape, device="cuda", generator=g).to(h.dtype)
    dl = torch.randn(last.shape, device="cuda", generator=g)
    grads = torch.autograd.grad((h, last), leaves, (dh, dl))
    want = so.scan(gate, x, h0, r, n, bf, dh, dl)
    for name, got in zip(("h", "last", "dgate", "dx", "dh0"), (h, last) + grads):
        assert got.dtype == (gate.dtype if name in ("h", "dgate", "dx") else torch.float32)
        so.within(got, *want[name], f"{what} {name}")
    with torch.no_grad():                                               # the same values without gradients
        h2, last2 = gated_scan(gate, x, h0, resets=r, lengths=n, batch_first=bf)
    assert torch.equal(h, h2) and torch.equal(last, last2)


@pytest.mark.parametrize("marks", ["none", "h0", "all"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,B,D", SHAPES)
def test_scan_matches_the_64_bit_form(torch_cuda, T, B, D, dtype, marks):
    torch = torch_cuda
    bf = (T + B + D) % 2 == 1
    gate, x, h0, r, n = _make(torch, T, B, D, getattr(torch, dtype), bf, T + D, marks == "all", marks == "all", marks != "none")
    _check(torch, gate, x, h0, r, n, bf, what=f"{T}x{B}x{D} {dtype} {marks}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scan_takes_strided_tensors(torch_cuda, dtype):
    torch = torch_cuda
    dt = getattr(torch, dtype)
    for T, B, D in ((50, 6, 24), (20, 300, 256), (11, 1200, 256)):
        both = torch.randn(T, B, 2 * D + 3, device="cuda").to(dt)      # one projection's output, cut in two
        _check(torch, both[..., :D], both[..., D + 3:], None, None, None, False, what="cut projection")
        _check(torch, both[..., 1:D + 1], both[..., D:2 * D], None, None, None, False, what="odd offset")
        _check(torch, both[..., :D].transpose(0, 1), both[..., :D].transpose(0, 1), None, None, None, True, what="transposed")
        one = torch.randn(T, 1, D, device="cuda").to(dt)                # a gate shared by all sequences
        _check(torch, one.expand(T, B, D), both[..., :D], None, torch.rand(1, B, device="cuda").expand(T, B) < 0.3, None, False, what="expanded")
        four = torch.randn(T, B, 2 * D + 4, device="cuda").to(dt)       # aligned rows, further apart than their length
        far0 = torch.randn(B * D + 1, device="cuda")[1:].view(B, D)     # a state that is aligned to nothing
        n = torch.randint(-3, T + 4, (B,), device="cuda", dtype=torch.int32)       # (lengths are clamped)
        _check(torch, four[..., :D], four[..., D:2 * D], far0, torch.rand(T, B, device="cuda") < 0.1, n, False, what="aligned cut")
        flat = torch.randn(1, 1, D, device="cuda").to(dt)               # one decay for all steps
        _check(torch, flat.expand(T, B, D), four[..., :D], far0, None, None, False, what="one gate")
        wide = torch.randn(T, B, 2 * D, device="cuda").to(dt)[..., ::2]  # last axis not contiguous: copied
        _check(torch, wide, wide, None, None, None, False, what="step of two")


def test_gradient_of_an_expanded_gate_sums(torch_cuda):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan
    T, B, D = 30, 5, 8
    one, x = torch.randn(T, 1, D, device="cuda", requires_grad=True), torch.randn(T, B, D, device="cuda")
    h, _ = gated_scan(one.expand(T, B, D), x)
    h.sum().backward()                                                  # (and an upstream gradient with all strides zero)
    want = so.scan(one.expand(T, B, D), x, dh=torch.ones(T, B, D))
    so.within(one.grad, want["dgate"][0].sum(1, keepdim=True), want["dgate"][1].sum(1, keepdim=True) + B * so.U * want["dgate"][0].abs().sum(1, keepdim=True), "gate")


def test_scan_gradients_against_differences(torch_cuda):
    """The gradients against central differences of the 64-bit form: truncation is of the order of step^2."""
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan
    T, B, D = 9, 2, 3
    gate, x, h0, r, n = _make(torch, T, B, D, torch.float32, False, 5, True, True, True)
    w, wl = torch.randn(T, B, D, device="cuda"), torch.randn(B, D, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (gate, x, h0)]
    h, last = gated_scan(*leaves, resets=r, lengths=n)
    ((h * w).sum() + (last * wl).sum()).backward()

    def value(k, e):
        args = [gate.double(), x.double(), h0.double()]
        args[k] = args[k] + e.view_as(args[k])
        gate64, x64, h64 = args
        hh, out = h64.cpu(), 0.0
        for t in range(T):
            kept = torch.where(r[t].cpu().unsqueeze(1), torch.zeros_like(hh), hh)
            new = torch.sigmoid(gate64[t].cpu()) * kept + torch.sigmoid(-gate64[t].cpu()) * x64[t].cpu()
            on = (t < n.cpu()).unsqueeze(1)
            out = out + (torch.where(on, new, torch.zeros_like(new)) * w[t].cpu().double()).sum()
            hh = torch.where(on, new, hh)
        return float(out + (hh * wl.cpu().double()).sum())

    step = 1e-4
    for k, leaf in enumerate(leaves):
        for j in range(leaf.numel()):
            e = torch.zeros(leaf.numel(), dtype=torch.float64, device="cuda")
            e[j] = step
            d = (value(k, e) - value(k, -e)) / (2 * step)
            # third derivatives of these sums stay below 1e3 at such values: 1e-8 x 1e3 / 6; float32 values of order 10: 1e-5
            assert abs(float(leaf.grad.reshape(-1)[j]) - d) <= 2e-6 + 1e-5 * max(1.0, abs(d)), (k, j)


def test_what_is_masked_is_not_read(torch_cuda):
    """NaN and infinities beyond the lengths and in front of a reset leave no trace; an empty sequence passes its state."""
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan
    for T, B, D in ((40, 6, 5), (40, 300, 256), (1500, 2, 4)):
        gate, x, h0, _, _ = _make(torch, T, B, D, torch.float32, False, 3, h0=True)
        n = torch.tensor([0, T, 1, T - 1, T // 2, 3] * (B // 6 + 1), device="cuda", dtype=torch.int32)[:B]
        r = torch.zeros(T, B, dtype=torch.bool, device="cuda")
        r[min(2, T - 1)] = True
        clean = [t.clone() for t in (gate, x, h0)]
        beyond = (torch.arange(T, device="cuda").unsqueeze(1) >= n)
        gate[beyond] = float("nan"); x[beyond] = float("inf")
        h0[n > 2] = float("inf")                                        # dropped by the reset, after two steps that show it
        dh = torch.randn(T, B, D, device="cuda"); dl = torch.randn(B, D, device="cuda")
        dirty = dh.clone(); dirty[beyond] = float("nan")
        L = [t.requires_grad_() for t in (gate, x)]
        h, last = gated_scan(*L, h0, resets=r, lengths=n)
        dg, dx = torch.autograd.grad((h, last), L, (dirty, dl))
        want = so.scan(clean[0], clean[1], clean[2], r, n, False, dh, dl)
        seen = torch.zeros(T, B, dtype=torch.bool, device="cuda"); seen[:2, n > 2] = True          # steps that see the infinite state
        ok = ~seen.cpu()
        for name, got in (("h", h), ("dgate", dg), ("dx", dx)):
            so.within(got.cpu()[ok], want[name][0][ok], want[name][1][ok], f"{name} {T}")
        so.within(last, *want["last"], f"last {T}")
        assert bool(torch.isinf(h[seen]).any())
        assert torch.equal(last[n == 0], h0[n == 0])


def test_gate_extremes(torch_cuda):
    """Gates at the ends of their type: the state is kept or replaced exactly; nothing becomes NaN."""
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan
    for dt in (torch.float32, torch.bfloat16):
        for big in (float("inf"), torch.finfo(dt).max, 200.0):
            gate = torch.tensor([big, -big, big, -big], device="cuda", dtype=dt).view(4, 1, 1).expand(4, 2, 3)
            x = torch.arange(1, 25, device="cuda").view(4, 2, 3).to(dt)
            h0 = torch.full((2, 3), 7.0, device="cuda")
            h, last = gated_scan(gate, x, h0)
            assert torch.equal(h[0], h0.to(dt)) and torch.equal(h[1], x[1]) and torch.equal(h[2], x[1]) and torch.equal(h[3], x[3])


def test_offsets_beyond_32_bits(torch_cuda):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan
    T, B, D = 3, 4, 64
    far = 2 ** 30 + 64
    big = torch.zeros(2 * far + B * D, device="cuda", dtype=torch.bfloat16)        # 4.3 GB
    gate = big.as_strided((T, B, D), (far, D, 1))
    src = torch.randn(T, B, D, device="cuda").to(torch.bfloat16)
    gate.copy_(src)
    x = torch.randn(T, B, D, device="cuda").to(torch.bfloat16)
    _check(torch, gate, x, None, None, None, False, what="far time steps")
    gb = big.as_strided((T, B, D), (D, far // 2, 1))                    # rows far apart
    gb.copy_(src)
    _check(torch, gb, x, None, None, None, False, what="far rows")
    del big


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("B,D", [(1, 1), (30, 64), (7, 61), (1025, 256)])
def test_step_is_the_scan_step_by_step(torch_cuda, B, D, dtype):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan, gated_scan_step
    dt, T = getattr(torch, dtype), 6
    gate, x, h0, r, _ = _make(torch, T, B, D, dt, False, B, resets=True, h0=True)
    want = so.scan(gate, x, h0, r)
    state, buf = h0.clone(), torch.empty(B, D + 4, device="cuda", dtype=dt)
    for t in range(T):
        v = state._version
        out = gated_scan_step(gate[t], x[t], state, reset=r[t], out=buf[:, 2:D + 2] if t % 2 else None)
        assert state._version > v
        so.within(out, want["h"][0][t], want["h"][1][t], f"step {t}")
    so.within(state, *want["last"], "state")
    h, last = gated_scan(gate, x, h0, resets=r)
    so.within(last, *want["last"], "scan's state")
    g = gate[0].clone()                                                 # in place over its own gate
    s1, s2 = h0.clone(), h0.clone()
    a = gated_scan_step(gate[0], x[0], s1)
    b = gated_scan_step(g, x[0], s2, out=g)
    assert b.data_ptr() == g.data_ptr() and torch.equal(a, b) and torch.equal(s1, s2)


ADV = [(1, 1, (1,)), (5, 3, (7,)), (33, 4, (1, 30)), (200, 40, (1, 30)), (333, 7, (13,)), (40, 2300, (30,)), (5000, 1, (3,)), (64, 64, ())]


@pytest.mark.parametrize("marks", ["none", "dones", "lengths", "both"])
@pytest.mark.parametrize("T,E,rest", ADV)
def test_advantages_match_the_64_bit_form(torch_cuda, T, E, rest, marks):
    torch = torch_cuda
    from marl_amd.recurrence import advantages
    g = torch.Generator(device="cuda").manual_seed(T + E)
    r = torch.randn(T, E, *rest, device="cuda", generator=g)
    v = torch.randn(T + 1, E, *rest, device="cuda", generator=g) * 3
    d = torch.rand(T, E, *rest, device="cuda", generator=g) < 0.05 if marks in ("dones", "both") else None
    n = torch.randint(0, T + 1, (E,), device="cuda", generator=g, dtype=torch.int32) if marks in ("lengths", "both") else None
    want = so.advantages(r, v, d, n, 0.97, 0.9)
    if n is not None:                                                   # what lies behind an end does not matter
        t = torch.arange(T + 1, device="cuda").view(T + 1, *([1] * (r.dim() - 1)))
        nn = n.view(1, E, *([1] * len(rest)))
        r = torch.where(t[:T] >= nn, torch.full_like(r, float("nan")), r)
        v = torch.where(t > nn, torch.full_like(v, float("nan")), v)
    adv, ret, mom = advantages(r, v, dones=d, lengths=n, gamma=0.97, lam=0.9, moments=True)
    adv2, ret2 = advantages(r, v, dones=d, lengths=n, gamma=0.97, lam=0.9)
    assert torch.equal(adv, adv2) and torch.equal(ret, ret2)
    so.within(adv, want[0], want[1], "adv")
    so.within(ret, want[2], want[3], "ret")
    # the moments: the elements' errors average at worst, one rounding; the deviation's error is at most that of its elements
    err = float(want[1].max())
    mean, sd = float(want[4]), float(want[5])
    assert abs(float(mom[0]) - mean) <= err + so.U * abs(mean) + 1e-12
    got_sd = 1.0 / float(mom[1]) - 1e-8
    assert abs(got_sd - sd) <= err + 4 * so.U * (sd + 1e-8) + 1e-7 * abs(mean)


def test_advantages_of_ring_slots_and_finished_episodes(torch_cuda):
    """Rings with time steps any distance apart; the value and the advantage behind a finished step do not count even when
    they are not finite."""
    torch = torch_cuda
    from marl_amd.recurrence import advantages
    T, E, n = 20, 6, 30
    ring = torch.randn(T, 3, E, 1, n, device="cuda")
    v = torch.randn(T + 1, 2, E, 1, n, device="cuda")
    d = torch.zeros(T, E, 1, n, dtype=torch.uint8, device="cuda")
    d[9] = 5
    want = so.advantages(ring[:, 1], v[:, 1], d, None)
    adv, ret = advantages(ring[:, 1], v[:, 1], dones=d)
    so.within(adv, want[0], want[1], "adv")
    v2 = v[:, 1].clone(); v2[10] = float("inf")
    r2 = ring[:, 1].clone(); r2[10:] = float("nan")
    adv2, ret2 = advantages(r2, v2, dones=d)
    assert torch.equal(adv2[:10], adv[:10]) and torch.equal(ret2[:10], ret[:10])


def test_captured_graphs_and_other_streams(torch_cuda, no_garbage):
    """Forward and backward in one HIP graph, replayed between eager work on other data; a second graph beside it; a side stream."""
    torch = torch_cuda
    from marl_amd.recurrence import advantages, gated_scan
    T, B, D = 600, 3, 20                                                # (the time axis is cut: a workspace is in use)
    mk = lambda: [torch.randn(T, B, D, device="cuda", requires_grad=True) for _ in range(2)]  # noqa: E731

    def work(L, dh):
        h, last = gated_scan(*L)
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), L, (dh, last.detach())) + \
            advantages(h.detach(), torch.cat((h.detach(), last.detach().unsqueeze(0))), moments=True)

    sets = [(mk(), torch.randn(T, B, D, device="cuda")) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            work(*s)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = work(*s)
        graphs.append((g, out))
    for k in range(3):
        with torch.no_grad():
            for L, dh in sets:
                for t in L:
                    t.copy_(torch.randn(T, B, D, device="cuda"))
                dh.copy_(torch.randn(T, B, D, device="cuda"))
        for g, _ in graphs:
            g.replay()
        for (g, out), s in zip(graphs, sets):
            eager = work(*s)
            assert all(torch.equal(a, b) for a, b in zip(out, eager)), k
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        other = work(*sets[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, work(*sets[0])))


def test_capture_beside_a_live_eager_graph_is_refused(torch_cuda, no_garbage):
    """The backward pass of such a capture would end the process: the call raises instead, before there is one."""
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    from marl_amd.recurrence import gated_scan
    gate, x = (torch.randn(4, 2, 8, device="cuda", requires_grad=True) for _ in range(2))
    std = torch.zeros(2, device="cuda", requires_grad=True)
    act, row = torch.randn(6, 2, device="cuda"), torch.randn(6, device="cuda")
    for call in (lambda: gated_scan(gate, x)[0], lambda: clipped_policy_loss(act, std, act, row, row)[0]):
        alive = call()
        with pytest.raises(RuntimeError, match="same leaf tensor"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        want = alive.detach().clone()
        del alive
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call().detach()
        g.replay()
        assert torch.equal(out, want)


def test_backward_notices_inputs_overwritten_since(torch_cuda):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan, gated_scan_step
    gate, x = (torch.randn(4, 2, 8, device="cuda", requires_grad=True) for _ in range(2))
    h0 = torch.zeros(2, 8, device="cuda")
    h, last = gated_scan(gate, x, h0)
    gated_scan_step(gate.detach()[0], x.detach()[0], h0)                # the rollout goes on with the same state
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    h, last = gated_scan(gate, x)
    last.sum().backward()                                               # only the last state has a gradient
    want = so.scan(gate, x, dlast=torch.ones(2, 8))
    so.within(gate.grad, *want["dgate"], "gate")
    so.within(x.grad, *want["dx"], "x")


def test_second_derivatives_are_refused(torch_cuda):
    torch = torch_cuda
    from marl_amd.policy_loss import clipped_policy_loss
    from marl_amd.recurrence import gated_scan
    gate, x = (torch.randn(4, 2, 8, device="cuda", requires_grad=True) for _ in range(2))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gated_scan(gate, x)[0].sum(), gate, create_graph=True)
    mean, row = torch.randn(6, 2, device="cuda", requires_grad=True), torch.randn(6, device="cuda")
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(clipped_policy_loss(mean, torch.zeros(2, device="cuda"), mean.detach(), row, row)[0], mean, create_graph=True)


@pytest.mark.parametrize("D", [64, 256])
def test_c_entries_take_sequences_in_reverse_order(torch_cuda, D):
    """Strides of the C entries may be negative: the batch, or time, read from its far end."""
    torch = torch_cuda
    from marl_amd import _lib
    lib, T, B = _lib.load(), 19, 500
    gate, x, dh = (torch.randn(T, B, D, device="cuda") for _ in range(3))
    cut = (torch.rand(T, B, device="cuda") < 0.1).to(torch.uint8)
    for axis in (0, 1):
        h, dgate, dx = (torch.zeros_like(gate) for _ in range(3))

        def at(t):
            s = list(t.stride()[:2])
            first = t.data_ptr() + (t.shape[axis] - 1) * s[axis] * t.element_size()
            s[axis] = -s[axis]
            return (first, *s)
        st = torch.cuda.current_stream().cuda_stream
        need = lib.asm_gated_scan_workspace(0, T, B, D)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        kept = lib.asm_gated_scan_kept(0, T, B, D)
        kept = torch.empty(kept, dtype=torch.uint8, device="cuda") if kept else None
        pk = None if kept is None else kept.data_ptr()
        _lib.check(lib.asm_gated_scan_forward(0, T, B, D, *at(gate), *at(x), None, *at(cut), None, *at(h), None, pk, ws.data_ptr(), need, st), "forward")
        _lib.check(lib.asm_gated_scan_backward(0, T, B, D, *at(gate), *at(x), *at(h), None, *at(cut), None, *at(dh), None, *at(dgate), *at(dx), None, pk,
                                               ws.data_ptr(), need, st), "backward")
        turned = lambda t: t.flip(axis)  # noqa: E731
        want = so.scan(turned(gate), turned(x), resets=turned(cut) != 0, dh=turned(dh))
        for name, got in (("h", h), ("dgate", dgate), ("dx", dx)):
            so.within(turned(got), *want[name], f"axis {axis} {name}")


def test_step_refuses_outputs_on_its_state(torch_cuda):
    torch = torch_cuda
    from marl_amd.recurrence import gated_scan_step
    gate, x, buf = torch.randn(6, 8, device="cuda"), torch.randn(6, 8, device="cuda"), torch.zeros(20, 8, device="cuda")
    for out in (buf[4:10], buf[9:15], buf.view(10, 16)[2:8, :8]):       # state: rows 4 to 9
        with pytest.raises(ValueError, match="share memory"):
            gated_scan_step(gate, x, buf[4:10], out=out)
    assert not buf.any()
    want = gated_scan_step(gate, x, torch.zeros(6, 8, device="cuda"))
    gated_scan_step(gate, x, buf[4:10], out=buf[10:16])                 # one buffer, different rows
    assert torch.equal(buf[10:16], want) and torch.equal(buf[4:10], want) and not buf[:4].any() and not buf[16:].any()
