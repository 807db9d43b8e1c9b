"""Outputs of the C entries that overlap each other or an input.  Runs on the CPU and on nothing else: the addresses are made up,
a call that is not refused fails at its launch for want of a device."""
import random

import pytest
import torch

from marl_amd import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses must not reach a device")
BASE = 1 << 30


def _bytes(p, elem, *axes):
    """Every byte of a strided tensor; axes: (count, stride in elements)."""
    at = [p]
    for n, s in axes:
        at = [a + i * s * elem for a in at for i in range(n)]
    return [a + k for a in at for k in range(elem)]


def _step(dtype, B, D, gate, x, state, reset, out):
    """Each of gate, x, out: (address, row stride); reset: the same or None.  Whether it was refused for an overlap."""
    lib = _lib.load()
    rc = lib.asm_gated_scan_step(dtype, B, D, gate[0], gate[1], x[0], x[1], state, reset[0] if reset else None, reset[1] if reset else 0, out[0], out[1], None)
    assert rc != 0
    return "share memory" in lib.asm_last_error().decode()


def test_step_by_hand():
    B, D, far = 6, 8, BASE + (1 << 20)
    for dtype, e in ((0, 4), (1, 2)):
        g, x, s, o = (BASE, D), (BASE + 4096, D), BASE + 8192, (BASE + 16384, D)
        ok = lambda *a: not _step(dtype, B, D, *a)  # noqa: E731
        assert ok(g, x, s, None, o) and ok(g, x, s, (far, 1), o)
        assert ok(g, x, s, None, g) and ok(g, x, s, None, x)            # out is gate or x itself
        assert ok(g, g, s, None, g)
        assert not ok(g, x, s, None, (g[0] + e, D)) and not ok(g, x, s, None, (g[0] - e, D)) and not ok(g, x, s, None, (x[0] + D * e, D))
        assert not ok((BASE, 0), x, s, None, g)                         # one gate for all rows, written by the first
        assert not ok(g, x, s, None, (s, D)) and not ok(g, x, s, None, (s + (B * D - 1) * 4, D)) and ok(g, x, s, None, (s + B * D * 4, D))
        assert ok((s, D), x, s, None, o) == (dtype == 0)                # the state is the gate: in float32 alone one layout
        assert not ok(g, x, s, (o[0] + 3, 1), o) and not ok(g, x, s, (s, 4), o) and ok(g, x, s, (s + B * D * 4, 1), o)
        w = 4 * D                                                       # one projection's output, cut in pieces
        assert ok((BASE, w), (BASE + D * e, w), s, None, (BASE + 2 * D * e, w)) and ok((BASE, w), (BASE + D * e, w), s, None, (BASE + 3 * D * e, w))
        assert not ok((BASE, w), (BASE + D * e, w), s, None, (BASE + (2 * D - 1) * e, w))
        assert not ok((BASE, w), (BASE + D * e, w), s, None, (BASE + (3 * D + 1) * e, w))
        assert ok((BASE, w), (BASE + D * e, w), s, (BASE + 2 * D * e, w * e), (BASE + 3 * D * e, w))


def test_step_against_every_byte():
    rng = random.Random(7)
    seen = [0, 0]
    for _ in range(3000):
        dtype, B, D = rng.randrange(2), rng.randrange(1, 5), rng.randrange(1, 5)
        e = 2 if dtype else 4
        place = lambda: BASE + e * rng.randrange(0, 60)  # noqa: E731
        gate, x, out = [(place(), rng.choice([D, D + 1, 2 * D, 3 * D, 7, -D, -9])) for _ in range(3)]
        gate = rng.choice([gate, (gate[0], 0), out])
        state = BASE + 4 * rng.randrange(0, 60)
        reset = rng.choice([None, None, (BASE + rng.randrange(0, 240), rng.choice([0, 1, 5]))])
        axes = lambda t: ((B, t[1]), (D, 1))  # noqa: E731
        G, X, O, S = _bytes(gate[0], e, *axes(gate)), _bytes(x[0], e, *axes(x)), _bytes(out[0], e, *axes(out)), _bytes(state, 4, (B * D, 1))
        R = _bytes(reset[0], 1, (B, reset[1])) if reset else []
        bad = bool(set(S) & set(O)) or bool(set(R) & (set(S) | set(O)))
        for to in (S, O):
            for frm in (G, X):
                bad = bad or (to != frm and bool(set(to) & set(frm)))
        if abs(out[1]) < D and B > 1:                                   # (rows of out that lie in each other)
            continue
        assert _step(dtype, B, D, gate, x, state, reset, out) == bad, (dtype, B, D, gate, x, state, reset, out)
        seen[bad] += 1
    assert min(seen) > 100, seen


def _act(dtype, B, n, A, mean, std, noise, actions, log_pi):
    """Each: (address, strides of the three axes); noise: the same or None."""
    import struct
    lib = _lib.load()
    rows = struct.pack("20q", *mean, *std, *(noise or (0, 0, 0, 0)), *actions, *log_pi)
    assert lib.asm_gaussian_act(dtype, B, n, A, rows, None) != 0
    return "share memory" in lib.asm_last_error().decode()


def test_actions_against_every_byte():
    rng = random.Random(11)
    seen = [0, 0]
    for _ in range(4000):
        dtype, B, n, A = rng.randrange(2), rng.randrange(1, 4), rng.randrange(1, 4), rng.randrange(1, 4)
        e = 2 if dtype else 4
        full = lambda: rng.choice([(n * A, A, 1), (n * A, 1, n), (3 * n * A, 3 * A, 1), (3 * n * A, 1, 3 * n), (n * A + 2, A, 1), (1, B, B * n), (-n * A, A, 1)])  # noqa: E731
        at = lambda elem: BASE + elem * rng.randrange(0, 70)  # noqa: E731
        mean, std, noise, act = (at(e), *full()), (at(e), *rng.choice([full(), (0, 0, 1)])), rng.choice([None, (at(4), *full())]), (at(4), *full())
        if noise and rng.random() < 0.3:
            act = rng.choice([noise, mean])
        lp = (at(4), *rng.choice([(n, 1), (3 * n, 3), (n + 1, 1), (1, B), (0, 1), (1, 1)]), 0)
        axes = lambda t: ((B, t[1]), (n, t[2]), (A, t[3]))  # noqa: E731
        M, S, U, L = _bytes(mean[0], e, *axes(mean)), _bytes(std[0], e, *axes(std)), _bytes(act[0], 4, *axes(act)), _bytes(lp[0], 4, (B, lp[1]), (n, lp[2]))
        N = _bytes(noise[0], 4, *axes(noise)) if noise else []
        bad = len(set(L)) < len(L) or bool(set(L) & (set(M) | set(S) | set(N) | set(U)))
        if noise:
            bad = bad or len(set(U)) < len(U)
            for frm in (M, S, N):
                bad = bad or (U != frm and bool(set(U) & set(frm)))
        assert _act(dtype, B, n, A, mean, std, noise, act, lp) == bad, (dtype, B, n, A, mean, std, noise, act, lp)
        seen[bad] += 1
    assert min(seen) > 100, seen
