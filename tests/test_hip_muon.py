"""Muon (csrc/muon_kernels.hip): the momentum, the Newton-Schulz orthogonalisation and the step against float64, and the refusals.

Tolerances, of the orthogonalised matrix in the Frobenius norm.  prec 3 holds every operand to 22 bits (2^-23 relative, half a step), prec 2
to 11 (2^-12).  A step rounds three operands; the relative error passes a step with at most |p'(s)| s / |p(s)| <= 1.6 once the singular values
are in the polynomial's interval and <= 1 before it.  15 roundings x 2.5: 5e-6 and (2^-12 / sqrt 3 x 15 x 2.5) 5e-3; the bounds are 1e-5 and
5e-3, plus the rounding of the output type (its half step)."""
import math
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "factored-neus_amd"))

C3 = (3.4445, -4.7750, 2.0315)
SIZES = [(1, 1), (1, 300), (2, 3), (39, 256), (64, 64), (63, 65), (256, 256), (217, 256), (512, 63), (144, 512), (256, 1), (129, 1000), (700, 640)]


def ns64(u, steps=5, eps=1e-7, coef=C3):
    a, b, c = coef
    x = u.double()
    x = x / max(float(x.norm()), eps)
    if x.shape[0] > x.shape[1]:
        return ns64(u.t(), steps, eps, coef).t()
    for _ in range(steps):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def matrix(rows, cols, seed=0, spread=0.7):
    g = torch.Generator().manual_seed(seed + 1000 * rows + cols)
    m = torch.randn(rows, cols, generator=g)
    return m * torch.exp(spread * (torch.randn(rows, 1, generator=g) + torch.randn(1, cols, generator=g))) * 1e-3


def bound(prec, t):
    return (1e-5 if prec == 3 else 5e-3) + torch.finfo(t).eps / 2


def off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_newton_schulz_against_float64(t, size):
    from fneus import ops
    g = (matrix(*size) * (100 if t == torch.float16 else 1)).to(t)
    want = ns64(g)
    for prec in (None, ops.PREC_PARITY, ops.PREC_H16):
        got = ops.newton_schulz(g.cuda(), prec=prec)
        assert got.dtype == t and got.shape == g.shape
        p = prec or (3 if t == torch.float32 else 2)
        assert off(got, want) <= bound(p, t), (prec, off(got, want))


@pytest.mark.gpu
def test_newton_schulz_large_and_stacked():
    """the 128-wide tiles, more matrices than one round of launches takes, every matrix as on its own, the same bits in every run"""
    from fneus import ops
    g = matrix(1537, 1800).cuda()
    want = ns64(g)
    got = ops.newton_schulz(g)
    assert off(got, want.cpu()) <= bound(3, torch.float32)
    assert torch.equal(ops.newton_schulz(g), got)
    got = ops.newton_schulz(g.t().contiguous())
    assert off(got, want.t().cpu()) <= bound(3, torch.float32)
    stack = torch.stack([matrix(40, 30, seed=k) for k in range(70)]).cuda()
    out = ops.newton_schulz(stack)
    for k in (0, 31, 32, 69):
        assert torch.equal(out[k], ops.newton_schulz(stack[k]))
        assert off(out[k], ns64(stack[k].cpu())) <= bound(3, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,t", [((3400, 3456), torch.float32), ((3456, 3400), torch.bfloat16), ((10, 1100, 1028), torch.float32)], ids=str)
def test_newton_schulz_shared_out(shape, t):
    """sizes whose symmetric products are shared out evenly and joined (105 tiles of one matrix; 150 of ten)"""
    from fneus import ops
    g = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).to(t).cuda()
    got = ops.newton_schulz(g)
    prec = 3 if t == torch.float32 else 2
    for k, (a, b) in enumerate([(got, g)] if g.dim() == 2 else [(got[0], g[0]), (got[9], g[9])]):
        want = ns64(b)
        err = float((a.double() - want).norm() / want.norm())
        assert err <= bound(prec, t), (k, err)
    assert torch.equal(ops.newton_schulz(g), got)


@pytest.mark.gpu
def test_muon_and_linear_on_two_streams_at_once():
    """two calls in flight: each has its own scratch and job table"""
    from fneus import ops
    gs = [torch.randn(8, 256, 256, device="cuda") for _ in range(2)]
    xs = [torch.randn(4096, 512, device="cuda") for _ in range(2)]
    w = torch.randn(512, 512, device="cuda")
    want = [(ops.newton_schulz(g), ops.linear_bwd(x, x, w)) for g, x in zip(gs, xs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, g, x in zip(streams, gs, xs):
            with torch.cuda.stream(s):
                got.append((ops.newton_schulz(g), ops.linear_bwd(x, x, w)))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(got, want):
            assert torch.equal(a, c) and all(torch.equal(p, q) for p, q in zip(b, d))


@pytest.mark.gpu
def test_newton_schulz_properties():
    """singular values in the polynomial's interval, the singular vectors kept; scale-free; other polynomials and step counts; zero, tiny,
    huge, rank-deficient and NaN matrices"""
    from fneus import ops
    g = matrix(96, 130).cuda()
    o = ops.newton_schulz(g)
    s = torch.linalg.svdvals(o.double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25
    for f in (2.0 ** 40, 2.0 ** -40):
        assert torch.equal(ops.newton_schulz(g * f, eps=1e-30), ops.newton_schulz(g, eps=1e-30))
    assert off(ops.newton_schulz(g * 1e30), ns64(g.cpu())) <= 2e-5           # |g|^2 beyond fp32's range
    for coef, steps in (((2.0, -1.5, 0.5), 1), ((1.875, -1.25, 0.375), 12), ((8.28, -23.6, 17.3), 1)):
        assert off(ops.newton_schulz(g, coefficients=coef, steps=steps), ns64(g.cpu(), steps, coef=coef)) <= 1e-5
    assert float(ops.newton_schulz(torch.zeros(20, 30, device="cuda")).abs().max()) == 0.0
    tiny = torch.full((4, 4), 1e-12, device="cuda")                           # below eps: divided by eps, not by the norm
    assert off(ops.newton_schulz(tiny), ns64(tiny.cpu())) <= 1e-5
    # rank 3: what rounding adds in the directions without a singular value grows by a^5 = 485, a^4 = 141, a^3 = 41, ... from the step it
    # enters at.  |X|_F is 1 at first and at most 1.2 sqrt 3 = 2.1 later, half a step of 22 bits is 2^-23 of it, |NS|_F >= 0.7 sqrt 3 = 1.2:
    # 2^-23 (485 + 2.1 (141 + 41 + 12 + 3.4 + 1)) / 1.2 = 9e-5 (fp32 arithmetic: half of it)
    low = (matrix(200, 3) @ matrix(3, 150)).cuda()
    assert off(ops.newton_schulz(low), ns64(low.cpu())) <= 9e-5
    bad = g.clone()
    bad[3, 4] = float("nan")
    assert bool(torch.isnan(ops.newton_schulz(bad)).all())
    assert ops.newton_schulz(g[:0]).shape == (0, 130)
    view = torch.randn(50, 40, device="cuda").t()
    assert torch.equal(ops.newton_schulz(view), ops.newton_schulz(view.contiguous()))


def step64(p, g, m, lr, mu, nesterov, wd, adj):
    m = mu * m.double() + (1 - mu) * g.double()
    u = (1 - mu) * g.double() + mu * m if nesterov else m
    return p.double() * (1 - lr * wd) - lr * adj * ns64(u), m


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_against_float64(nesterov):
    from fneus import ops
    sizes = [(256, 256), (512, 63), (144, 512), (512, 512), (3, 1), (256, 90)]
    ps, gs, ms = ([matrix(*s, seed=k).cuda() for s in sizes] for k in (1, 2, 3))
    want = []
    for p, g, m in zip(ps, gs, ms):
        adj = ops.muon_adjust("original", *p.shape)
        want.append(step64(p.cpu(), g.cpu(), m.cpu(), 0.03, 0.9, nesterov, 0.1, adj))
    lr = torch.full((), 0.03, device="cuda")
    ops.muon_step(ps, gs, ms, lr, momentum=0.9, nesterov=nesterov, weight_decay=0.1, adjust="original", zero_grad=True)
    for (wp, wm), p, m, g in zip(want, ps, ms, gs):
        assert off(m, wm) <= 4 * 2.0 ** -24
        assert off(p, wp) <= 1e-5 + 4 * 2.0 ** -24
        assert float(g.abs().max()) == 0.0
    assert abs(ops.muon_adjust("match_rms", 4, 100) - 2.0) < 1e-12 and ops.muon_adjust(0.5, 3, 3) == 0.5


@pytest.mark.gpu
def test_muon_step_sixteen_bits_and_frozen_gradients():
    from fneus import ops
    for t in (torch.bfloat16, torch.float16):
        p, g, m = (matrix(120, 200, seed=k).mul(200).to(t).cuda() for k in (1, 2, 3))
        keep = g.clone()
        p0, m0 = p.cpu(), m.cpu()
        ops.muon_step([p], [g], [m], 0.02, adjust=1.0)
        assert torch.equal(g, keep)
        wm = (0.95 * m0.double() + (1 - 0.95) * keep.cpu().double())
        assert off(m, wm) <= torch.finfo(t).eps / 2 + 1e-6
        wp = p0.double() - 0.02 * ns64((1 - 0.95) * keep.cpu().double() + 0.95 * m.cpu().double())
        assert off(p, wp) <= 5e-3 + torch.finfo(t).eps / 2


@pytest.mark.gpu
def test_muon_step_in_a_graph():
    """replayed with new gradients and a new learning rate between the replays, against the eager step"""
    from fneus import ops
    sizes = [(256, 256), (100, 60), (512, 144)]
    ps, gs, ms = ([matrix(*s, seed=k).cuda() for s in sizes] for k in (1, 2, 3))
    lr = torch.full((), 0.02, device="cuda")
    pe, me = [p.clone() for p in ps], [m.clone() for m in ms]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.muon_step(ps, gs, ms, lr)
    torch.cuda.current_stream().wait_stream(side)
    ops.muon_step(pe, gs, me, lr)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_step(ps, gs, ms, lr)
    for k in range(3):
        for g in gs:
            g.copy_(torch.randn_like(g))
        lr.fill_(0.01 / (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        ops.muon_step(pe, gs, me, lr)
        assert all(torch.equal(a, b) for a, b in zip(ps + ms, pe + me)), k


def test_muon_refusals_cpu():
    import ctypes as C
    from fneus import ops
    from fneus._lib import lib, FneusMuonJob
    with pytest.raises(ValueError):
        ops.newton_schulz(torch.randn(3, 3))
    with pytest.raises(ValueError):
        ops.muon_step([torch.randn(3, 3)], [torch.randn(3, 3)], [torch.randn(3, 3)], 0.1)
    ops.muon_step([], [], [], 0.1)
    jobs = (FneusMuonJob * 1)()
    jobs[0].grad, jobs[0].out, jobs[0].rows, jobs[0].cols = 256, 256, 4, 4
    need = lib.fneus_muon_scratch_bytes(jobs, 1, 3)
    assert need > 0 and need > lib.fneus_muon_scratch_bytes(jobs, 1, 2)
    ns = lambda coef=C3, steps=5, eps=1e-7, prec=3, dtype=0, scratch=256, n=None, jobs=jobs: lib.fneus_newton_schulz(  # noqa: E731
        jobs, 1, *coef, steps, eps, prec, dtype, C.c_void_p(scratch), need if n is None else n, None)
    for k in (dict(steps=0), dict(steps=65), dict(eps=0.0), dict(prec=1), dict(dtype=3), dict(scratch=None), dict(scratch=264), dict(n=need - 1),
              dict(coef=(9.0, 9.0, 9.0)), dict(coef=(float("nan"), 1.0, 1.0))):
        assert ns(**k) == -2, k
    for field, value in (("rows", 0), ("cols", -1), ("rows", 70000), ("grad", None), ("out", None)):
        bad = (FneusMuonJob * 1)()
        bad[0].grad, bad[0].out, bad[0].rows, bad[0].cols = 256, 256, 4, 4
        setattr(bad[0], field, value)
        assert ns(jobs=bad, n=1 << 40) == -2, field
    assert lib.fneus_muon(jobs, 1, C.c_void_p(256), 0.9, 1, 0.0, *C3, 5, 1e-7, 3, 0, 0, C.c_void_p(256), need, None) == -2      # no momentum, no parameter


@pytest.mark.gpu
def test_muon_refusals():
    from fneus import ops
    p, g, m = (torch.randn(6, 5, device="cuda") for _ in range(3))
    for bad in (lambda: ops.muon_step([p], [g[:5]], [m], 0.1), lambda: ops.muon_step([p], [g], [], 0.1), lambda: ops.muon_step([p], [p], [m], 0.1),
                lambda: ops.muon_step([p[0]], [g[0]], [m[0]], 0.1), lambda: ops.muon_step([p], [g.half()], [m], 0.1),
                lambda: ops.muon_step([p.t()], [g.t()], [m.t()], 0.1), lambda: ops.muon_step([p, p], [g, m], [m, g], 0.1),
                lambda: ops.muon_step([p[:4], p[2:]], [g[:4], g[:4].clone()], [m[:4], m[:4].clone()], 0.1),
                lambda: ops.muon_step([p], [g], [m], torch.ones(2, device="cuda")), lambda: ops.muon_step([p], [g], [m], 0.1, adjust="other"),
                lambda: ops.muon_step([p], [g], [m], 0.1, prec=1), lambda: ops.newton_schulz(p.double()), lambda: ops.newton_schulz(p[0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.newton_schulz(p, steps=0)


# A side of at most 64: three launches in fp64.  What is left is the rounding of the output: half a step of its type (fp16: of its subnormal
# values, 2^-25, each), and fp64's of u u^T (2^-53 sqrt(n)) grown by 11.9^4 = 2e4: below 1e-9 for n <= 2^16; 1e-7 covers the fp32 in between.
def few_bound(t, want):
    return torch.finfo(t).eps / 2 + 1e-7 + (2.0 ** -25 * want.numel() ** 0.5 / float(want.norm()) if t == torch.float16 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [(1, 1), (1, 64), (64, 1), (5, 5), (16, 129), (17, 128), (127, 32), (33, 40), (48, 1000), (63, 64), (64, 64), (640, 64),
                                  (64, 20001), (9999, 15), (2, 65536)], ids=str)
def test_newton_schulz_of_a_short_side(t, size):
    from fneus import ops
    g = (matrix(*size) * (100 if t == torch.float16 else 1)).to(t)
    want = ns64(g)
    for prec in (ops.PREC_PARITY, ops.PREC_H16):
        assert off(ops.newton_schulz(g.cuda(), prec=prec), want) <= few_bound(t, want)


@pytest.mark.gpu
def test_newton_schulz_of_a_short_side_properties():
    """step counts and polynomials on both sides of the rule for the form; rank-deficient, zero, tiny, huge, NaN matrices; a stack"""
    from fneus import ops
    g = matrix(40, 90).cuda()
    for coef, steps in ((C3, 1), (C3, 2), (C3, 7), ((2.0, -1.5, 0.5), 3), ((1.875, -1.25, 0.375), 12), ((8.28, -23.6, 17.3), 1)):
        want = ns64(g.cpu(), steps, coef=coef)
        assert off(ops.newton_schulz(g, coefficients=coef, steps=steps), want) <= few_bound(torch.float32, want)
    low = (matrix(60, 2) @ matrix(2, 50)).cuda()
    for steps in (5, 7, 8, 30):                 # (from 8 steps on an error of A has room to grow: the tiled form)
        s = torch.linalg.svdvals(ops.newton_schulz(low, steps=steps).double())
        assert bool(torch.isfinite(s).all()) and float(s[0]) < 1.25
    # rank 2 but for the entries' own fp32 rounding, which the same fp64 polynomial amplifies in both
    assert off(ops.newton_schulz(low), ns64(low.cpu())) <= few_bound(torch.float32, ns64(low.cpu()))
    assert float(ops.newton_schulz(torch.zeros(20, 30, device="cuda")).abs().max()) == 0.0
    for f in (2.0 ** 40, 2.0 ** -40):
        assert torch.equal(ops.newton_schulz(g * f, eps=1e-30), ops.newton_schulz(g, eps=1e-30))
    assert off(ops.newton_schulz(g * 1e34), ns64(g.cpu())) <= 1e-6          # (g 1e34: a rounding of every entry)
    bad = g.clone()
    bad[3, 4] = float("nan")
    assert bool(torch.isnan(ops.newton_schulz(bad)).all())
    stack = torch.stack([matrix(30, 70, seed=k) for k in range(70)]).cuda()
    out = ops.newton_schulz(stack)
    for k in (0, 31, 32, 69):
        assert torch.equal(out[k], ops.newton_schulz(stack[k]))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_muon_of_short_and_long_sides_together(t):
    """more matrices of each form than a round of launches takes, in one call; gradients cleared, neighbours in memory left alone"""
    from fneus import ops
    sizes = [((7 + k, 300 - k) if k % 2 else (70 + k, 66 + k)) if k % 3 else (130 + k, 5 + k // 2) for k in range(80)]
    n = sum(r * c + 1 for r, c in sizes)
    arenas = [torch.full((n,), 7.0, dtype=t, device="cuda") for _ in range(3)]
    sets, at = ([], [], []), 0
    for r, c in sizes:
        for k, (arena, out) in enumerate(zip(arenas, sets)):
            out.append(arena[at:at + r * c].view(r, c))
            out[-1].copy_(matrix(r, c, seed=k).mul(100))
        at += r * c + 1
    ps, gs, ms = sets
    p0, g0, m0 = ([x.cpu().clone() for x in s] for s in sets)
    lr = torch.full((), 0.03, device="cuda")
    ops.muon_step(ps, gs, ms, lr, momentum=0.9, weight_decay=0.1, adjust=1.0, zero_grad=True)
    prec, half = (3 if t == torch.float32 else 2), torch.finfo(t).eps / 2
    f, lr = torch.float32, 0.03
    for k in range(len(sizes)):
        m1 = ms[k].cpu()
        # (three fp32 roundings in front of the one to t)
        assert off(m1, 0.9 * m0[k].double() + (1 - 0.9) * g0[k].double()) <= half + 4 * 2.0 ** -24
        u = (1 - 0.9) * g0[k].double() + 0.9 * m1.double()
        want = p0[k].double() * (1 - lr * 0.1) - lr * ns64(u)
        err = lr * bound(prec, f) * float(ns64(u).norm()) / float(want.norm())
        assert off(ps[k], want) <= half + 4 * 2.0 ** -24 + err, sizes[k]
        assert float(gs[k].abs().max()) == 0.0
    at = 0
    for r, c in sizes:
        at += r * c + 1
        assert all(float(a[at - 1]) == 7.0 for a in arenas)


@pytest.mark.gpu
def test_muon_of_a_short_side_in_a_graph():
    """replayed with new gradients and learning rates and eager work in between, against the eager step, bit for bit"""
    from fneus import ops
    sizes = [(64, 300), (40, 17), (1000, 33), (128, 128)]
    ps, gs, ms = ([matrix(*s, seed=k).cuda() for s in sizes] for k in (1, 2, 3))
    pe, me = [p.clone() for p in ps], [m.clone() for m in ms]
    lr = torch.full((), 0.02, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.muon_step(ps, gs, ms, lr)
    torch.cuda.current_stream().wait_stream(side)
    for dst, src in zip(ps + ms, pe + me):
        dst.copy_(src)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_step(ps, gs, ms, lr)
    for k in range(4):
        for g, s in zip(gs, sizes):
            g.copy_(matrix(*s, seed=10 + k))
        lr.fill_(0.01 * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        ops.muon_step(pe, gs, me, lr)
        for a, b in zip(ps + ms, pe + me):
            assert torch.equal(a, b)


# X X^T of a few long rows: its contraction shared out over the CUs
@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(1, 130, 5000), (1, 2975, 422), (3, 65, 3001), (1, 4160, 66), (2, 1500, 257), (1, 100, 30000)], ids=str)
def test_newton_schulz_of_long_rows(t, size):
    from fneus import ops
    count, rows, cols = size
    g = torch.stack([matrix(rows, cols, seed=k) for k in range(count)]).to(t)
    out = ops.newton_schulz(g.cuda())
    again = ops.newton_schulz(g.cuda())
    assert torch.equal(out, again)
    for k in range(count):
        assert off(out[k], ns64(g[k])) <= bound(3 if t == torch.float32 else 2, t)
