"""The linear layer with bias, activation and residual (csrc/linear_kernels.hip) against float64, forward, backward and its refusals.

Tolerances, per element, with S = |x| |W|^T + |b| (or the product's own operands) in 64 bits:
  rounding of the output          eps(t) / 2 |value|
  fp32 sums of K terms            (4 + 2 sqrt(K)) 2^-23 S       (K roundings of at most 2^-24 of partial sums <= S, as a random walk, with margin 4;
                                                                 the three-term form of fp32 drops 2^-24 of each product)
  delta rounded to 16 bits        eps(t) / 2 of sum |delta| |W|  (a bf16 / fp16 operand of the backward's products: every term half a step)
  the activation                  4 x 2^-23 |z| + its slope (<= 1.13) times the error of z
The backward is compared with the formula at the z it is given."""
import math
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "factored-neus_amd"))

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "leaky", "sigmoid", "softplus", "gelu", "silu"]
# (rows, n_in, n_out): one row, the row kernel's last row and the first beyond it, one value, odd sizes, a tile's edges, the tiled kernel's
# sizes on and off its borders, a long contraction of few columns (split) and few rows with a long contraction, many rows of a few values
SIZES = [(1, 1, 1), (1, 512, 144), (1, 4099, 70), (3, 7, 5), (16, 256, 256), (17, 90, 256), (33, 63, 129), (100, 512, 512), (257, 31, 64),
         (300, 65, 33), (640, 512, 384), (1000, 777, 1111), (2048, 256, 256), (1025, 520, 1032), (5000, 40, 24), (20000, 256, 128), (64, 4096, 96),
         (40000, 256, 1), (5000, 3, 257), (30000, 5, 3), (2000, 1, 1)]


def act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "leaky": lambda: torch.where(z > 0, z, 0.2 * z), "sigmoid": lambda: torch.sigmoid(z),
            "softplus": lambda: torch.logaddexp(torch.zeros_like(z), 100 * z) / 100, "gelu": lambda: z * 0.5 * torch.special.erfc(-z * math.sqrt(0.5)),
            "silu": lambda: z * torch.sigmoid(z)}[act]()


def dact64(z, act):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "leaky": lambda: torch.where(z > 0, 1.0, 0.2).double(),
            "sigmoid": lambda: s * (1 - s), "softplus": lambda: torch.sigmoid(100 * z),
            "gelu": lambda: 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
            "silu": lambda: s * (1 + z * (1 - s))}[act]()


def inputs(rows, n_in, n_out, t, seed=0):
    g = torch.Generator().manual_seed(seed + rows + 3 * n_in + 5 * n_out)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [v.to(t).cuda() for v in (r(rows, n_in), r(n_out, n_in) / math.sqrt(n_in), 0.3 * r(n_out), r(rows, n_out), r(rows, n_out))]


def check(got, want, lim, what):
    err = (got.double() - want).abs()
    bad = ~(err <= lim)
    assert not bool(bad.any()), (what, float((err / lim.clamp(min=1e-300)).max()), int(bad.sum()), got.shape)


def half(t):
    return torch.finfo(t).eps / 2 * 1.01


def sums(k):
    return (4 + 2 * math.sqrt(k)) * 2.0 ** -23


def forward_and_backward(rows, n_in, n_out, t, act, res, bias=True, need=(True, True, True)):
    from fneus import ops
    x, w, b, r, dy = inputs(rows, n_in, n_out, t)
    b, r = (b if bias else None), (r if res else None)
    y, z = ops.linear_fwd(x, w, b, act=act, residual=r, train=True)
    assert (z is None) == (act == "none") and y.dtype == t
    xd, wd = x.double(), w.double()
    zd, S = xd @ wd.t(), xd.abs() @ wd.t().abs()
    if bias:
        zd, S = zd + b.double(), S + b.double().abs()
    ez = sums(n_in) * S
    want = act64(zd, act)
    lim = 1.13 * ez + 4 * 2.0 ** -23 * (zd.abs() + want.abs())
    if res:
        want = want + r.double()
        lim = lim + 2.0 ** -23 * want.abs()
    check(y, want, lim + half(t) * (want.abs() + lim) + torch.finfo(t).smallest_normal, "y")
    if z is not None:
        check(z, zd, ez + half(t) * (zd.abs() + ez) + torch.finfo(t).smallest_normal, "z")
    dx, dw, db = ops.linear_bwd(dy, x, w, z, act=act, need=need)
    d = dy.double() * (dact64(z.double(), act) if z is not None else 1.0)
    # the derivative in fp32: exp / erf to a few 2^-24, and softplus' argument 100 z
    ed = dy.double().abs() * 8 * 2.0 ** -23 * (1 + (100 * z.double().abs()).clamp(max=20) * (act == "softplus") if z is not None else 1)
    op = d.abs() * half(t) * (t != torch.float32) + ed
    tiny = torch.finfo(t).smallest_normal
    for got, want, lim, k, what in ((dx, d @ wd, (op @ wd.abs()), n_out, "dx"), (dw, d.t() @ xd, (op.t() @ xd.abs()), rows, "dw"),
                                    (db, d.sum(0), ed.sum(0), rows, "db")):
        if got is None:
            continue
        total = {"dx": d.abs() @ wd.abs(), "dw": d.abs().t() @ xd.abs(), "db": d.abs().sum(0)}[what]
        lim = lim + sums(k) * total
        flush = 2.0 ** -25 * {"dx": wd.abs().sum(0)[None, :], "dw": xd.abs().sum(0)[None, :], "db": torch.zeros_like(want)}[what] * (t == torch.float16)
        check(got, want, lim + half(t) * (want.abs() + lim) + tiny + flush, what)      # (fp16: delta below its normal range, half a step of 2^-24)
    assert [g is not None for g in (dx, dw, db)] == list(need)
    return y, z, dx, dw, db


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_sizes(t, size):
    forward_and_backward(*size, t, "gelu", True)
    forward_and_backward(*size, t, "none", False)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("size", [(5, 70, 40), (200, 130, 77), (640, 512, 384)], ids=str)
def test_linear_activations(t, act, size):
    forward_and_backward(*size, t, act, False, bias=False)
    forward_and_backward(*size, t, act, True)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", [(9, 40, 24), (150, 66, 130), (4096, 256, 256)], ids=str)
def test_linear_each_gradient_alone(t, size):
    full = forward_and_backward(*size, t, "silu", False)[2:]
    for k in range(3):
        got = forward_and_backward(*size, t, "silu", False, need=tuple(i == k for i in range(3)))[2:]
        assert torch.equal(got[k], full[k])


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", [(7, 96, 40), (130, 96, 72), (3000, 256, 192)], ids=str)
def test_linear_views_and_repeats(t, size):
    """row strides, unaligned starts, transposed and broadcast views: the same values; the same bits in every run"""
    from fneus import ops
    rows, n_in, n_out = size
    x, w, b, r, dy = inputs(*size, t)
    y, z = ops.linear_fwd(x, w, b, act="silu", residual=r, train=True)
    g = ops.linear_bwd(dy, x, w, z, act="silu")
    wide = lambda v, pad: torch.cat([torch.full_like(v[:, :1], 7.0), v, v[:, :pad]], 1)[:, 1:1 + v.shape[1]]  # noqa: E731
    xs, rs, ds = wide(x, 6), wide(r, 3), wide(dy, 5)
    for xv, rv, dv in ((xs, rs, ds), (x.t().contiguous().t(), r.t().contiguous().t(), dy.t().contiguous().t())):
        y2, z2 = ops.linear_fwd(xv, w, b, act="silu", residual=rv, train=True)
        g2 = ops.linear_bwd(dv, xv, w, z2, act="silu")
        for p, q in zip((y2, z2) + g2, (y, z) + g):
            scale = float(q.double().abs().max())
            assert float((p.double() - q.double()).abs().max()) <= scale * (2 * torch.finfo(t).eps + 2e-5)
        assert torch.equal(ops.linear_fwd(xv, w, b, act="silu", residual=rv)[0], y2)
    y3, _ = ops.linear_fwd(x, w, b, act="silu", residual=r)
    assert torch.equal(y3, y)
    assert all(torch.equal(p, q) for p, q in zip(ops.linear_bwd(dy, x, w, z, act="silu"), g))
    one = dy[:1].expand(rows, n_out)
    assert all(torch.equal(p, q) for p, q in zip(ops.linear_bwd(one, x, w, z, act="silu"), ops.linear_bwd(one.contiguous(), x, w, z, act="silu")))


@pytest.mark.gpu
def test_linear_and_layer_norm_beyond_32_bits():
    """rows 16 MiB apart (the tiled kernel's loads have 32-bit offsets within a tile: such rows are copied), and arrays of more than 2^32 bytes"""
    from fneus import ops
    w = torch.randn(256, 256, device="cuda").bfloat16()
    far = torch.zeros(300 * ((1 << 23) + 8), dtype=torch.bfloat16, device="cuda").as_strided((300, 256), ((1 << 23) + 8, 1))
    far.copy_(torch.randn(300, 256, device="cuda"))
    near = far.contiguous()
    wide = torch.cat([w] * 16)                                      # (large enough for the tiled form)
    assert torch.equal(ops.linear_fwd(far, wide)[0], ops.linear_fwd(near, wide)[0])
    dy = torch.randn(300, 4096, device="cuda").bfloat16()
    assert all(torch.equal(a, b) for a, b in zip(ops.linear_bwd(dy, far, wide), ops.linear_bwd(dy, near, wide)))
    assert torch.equal(ops.layer_norm_fwd(far)[0], ops.layer_norm_fwd(near)[0])
    del far
    rows = (1 << 24) + 300                                          # x 256 x 2 bytes = 8 GiB
    x = torch.empty(rows, 256, dtype=torch.bfloat16, device="cuda")
    x[-300:] = near
    x[:-300] = 0
    y, z = ops.linear_fwd(x, w, act="silu", train=True)
    ref = ops.linear_fwd(near, w, act="silu", train=True)
    lim = 2 * torch.finfo(torch.bfloat16).eps * float(ref[0].abs().max())
    assert float((y[-300:].float() - ref[0].float()).abs().max()) <= lim and float(y[:-300].abs().max()) == 0.0
    n, mean, rstd = ops.layer_norm_fwd(x)
    assert torch.equal(n[-300:], ops.layer_norm_fwd(near)[0])
    dx, dw, db = ops.linear_bwd(y, x, w, z, act="silu")
    small = ops.linear_bwd(ref[0], near, w, ref[1], act="silu")
    for a, b in ((dx[-300:], small[0]), (dw, small[1]), (db, small[2])):
        assert float((a.float() - b.float()).abs().max()) <= 4 * torch.finfo(torch.bfloat16).eps * float(b.float().abs().max())
    dl = ops.layer_norm_bwd(x, x, None, mean, rstd)[0]
    assert float((dl[-300:].float() - ops.layer_norm_bwd(near, near, None, mean[-300:], rstd[-300:])[0].float()).abs().max()) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(6, 64, 48), (200, 96, 80), (2048, 512, 512)], ids=str)
def test_linear_nan_stays_in_its_row(size):
    from fneus import ops
    x, w, b, r, _ = inputs(*size, torch.float32)
    for t in TYPES:
        xt, wt, bt, rt = (v.to(t) for v in (x, w, b, r))
        clean = ops.linear_fwd(xt, wt, bt, act="relu", residual=rt)[0]
        bad = xt.clone()
        bad[3, 5], bad[1, 0] = float("nan"), float("inf")
        y = ops.linear_fwd(bad, wt, bt, act="none", residual=rt)[0]
        assert bool(torch.isnan(y[3]).all()) and not bool(torch.isfinite(y[1]).any())
        yr = ops.linear_fwd(bad, wt, bt, act="relu", residual=rt)[0]
        keep = [k for k in range(size[0]) if k not in (1, 3)]
        assert torch.equal(yr[keep], clean[keep]) and bool(torch.isnan(yr[3]).all())


@pytest.mark.gpu
def test_linear_gradient_against_differences():
    """<dL/dx, v> against (L(x + h v) - L(x - h v)) / 2h in 64 bits, through the kernel's own forward values in fp32"""
    from fneus import ops
    x, w, b, r, dy = inputs(40, 48, 56, torch.float32)
    for act in ("sigmoid", "gelu", "silu", "softplus"):
        y, z = ops.linear_fwd(x, w, b, act=act, residual=r, train=True)
        dx, dw, db = ops.linear_bwd(dy, x, w, z, act=act)
        loss = lambda xx, ww, bb: float((act64(xx @ ww.t() + bb, act) * dy.double()).sum())  # noqa: E731
        h = 1e-6
        for grad, which in ((dx, 0), (dw, 1), (db, 2)):
            args = [x.double(), w.double(), b.double()]
            v = torch.randn(grad.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64).cuda()
            up, dn = list(args), list(args)
            up[which], dn[which] = args[which] + h * v, args[which] - h * v
            num = (loss(*up) - loss(*dn)) / (2 * h)
            ref = float((grad.double() * v).sum())
            scale = float((grad.double().abs() * v.abs()).sum())
            assert abs(num - ref) <= 1e-5 * scale, (act, which, num, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_linear_graph_and_no_rows(t):
    from fneus import ops
    for size in ((200, 130, 77), (2048, 512, 512)):
        x, w, b, r, dy = inputs(*size, t)
        def run():
            y, z = ops.linear_fwd(x, w, b, act="gelu", residual=r, train=True)
            return (y, z) + ops.linear_bwd(dy, x, w, z, act="gelu")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        for k in range(3):
            x.copy_(torch.randn(x.shape, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, run())), k
    y, z = ops.linear_fwd(x[:0], w, b, act="gelu", residual=r[:0], train=True)
    assert y.shape == (0, 512)
    dx, dw, db = ops.linear_bwd(dy[:0], x[:0], w, z, act="gelu")
    assert dx.shape == (0, 512) and float(dw.abs().max()) == 0.0 and float(db.abs().max()) == 0.0


def test_linear_abi_refusals_cpu():
    import ctypes as C
    from fneus._lib import lib, FneusLinear
    ok = dict(x=64, weight=64, y=64, rows=0, ldx=8, n_in=8, n_out=8, act=0, dtype=0)
    fwd = lambda **k: lib.fneus_linear_fwd(C.byref(FneusLinear(**dict(ok, **k))), None)  # noqa: E731
    assert fwd() == 0                                                # no rows: nothing is launched
    for k in (dict(rows=-1), dict(n_in=0), dict(n_out=0), dict(act=7), dict(act=-1), dict(dtype=3), dict(rows=4, x=None), dict(rows=4, weight=None),
              dict(rows=4, y=None), dict(rows=4, ldx=7), dict(rows=4, residual=64, ld_residual=7), dict(rows=1 << 31), dict(n_in=1 << 23)):
        assert fwd(**k) == -2, k
    okb = dict(ok, rows=4, dy=64, lddy=8, dx=64, dweight=64, dbias=64)
    bwd = lambda **k: lib.fneus_linear_bwd(C.byref(FneusLinear(**dict(okb, **k))), None)  # noqa: E731
    for k in (dict(rows=0), dict(dy=None), dict(lddy=7), dict(act=1), dict(weight=None), dict(x=None), dict(ldx=7),
              dict(dx=None, dweight=None, dbias=None)):
        assert bwd(**k) == -2, k
    assert lib.fneus_linear_fwd(None, None) == -2


def test_linear_refusals_cpu():
    from fneus import ops
    x = torch.randn(4, 8)
    with pytest.raises(ValueError):
        ops.linear_fwd(x, torch.randn(3, 8))
    with pytest.raises(ValueError):
        ops.linear_fwd(x, torch.randn(3, 8), act="tanh")


@pytest.mark.gpu
def test_linear_refusals():
    from fneus import ops
    x, w, b, r, dy = inputs(4, 8, 6, torch.float32)
    for bad in (lambda: ops.linear_fwd(x, w[:, :7]), lambda: ops.linear_fwd(x, w.half()), lambda: ops.linear_fwd(x, w, b.half()),
                lambda: ops.linear_fwd(x, w, b[:5]), lambda: ops.linear_fwd(x, w, b, residual=r[:, :5]), lambda: ops.linear_fwd(x, w, b, act=7),
                lambda: ops.linear_fwd(x[0], w), lambda: ops.linear_fwd(x.double(), w.double()), lambda: ops.linear_fwd(x, w.cpu()),
                lambda: ops.linear_bwd(dy, x, w, None, act="gelu"), lambda: ops.linear_bwd(dy[:3], x, w), lambda: ops.linear_bwd(dy.half(), x, w),
                lambda: ops.linear_fwd(x, w[:0])):
        with pytest.raises(ValueError):
            bad()


# Heads: up to 16 outputs (their own form each way), on both sides of the rules for it and of its blocks: 64 rows, lanes of 4 columns, strips of
# 1024 columns, the last four columns shared; more parts than one
HEADS = [(1025, 16, 1), (1024, 64, 8), (1100, 17, 4), (3000, 63, 5), (2049, 257, 3), (5000, 1031, 8), (9000, 4100, 2), (70001, 18, 7), (33000, 260, 16),
         (40000, 41, 9), (8200, 300, 16), (100, 5001, 16), (17, 300, 12), (1026, 15, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", HEADS, ids=str)
def test_linear_heads(t, size):
    forward_and_backward(*size, t, "sigmoid", True)
    forward_and_backward(*size, t, "none", False, bias=False)


@pytest.mark.gpu
@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (True, True, False), (False, True, True),
                                  (True, False, True)], ids=str)
def test_linear_heads_one_gradient_at_a_time(need):
    for size in ((3000, 90, 3), (3000, 1500, 8), (34000, 100, 16)):
        forward_and_backward(*size, torch.bfloat16, "silu", False, need=need)


@pytest.mark.gpu
@pytest.mark.parametrize("t", TYPES)
def test_linear_heads_strided_rows_and_neighbours(t):
    """rows apart, unaligned starts; nothing outside the outputs is written; the same bits twice; an infinite x stays in its own row and column"""
    from fneus import ops
    rows, n_in, n_out = 3001, 517, 6
    x, w, b, r, dy = inputs(rows, n_in, n_out, t)
    wide = torch.zeros(rows, n_in + 9, dtype=t, device="cuda")
    wide[:, 3:3 + n_in] = x
    dwide = torch.zeros(rows, n_out + 5, dtype=t, device="cuda")
    dwide[:, 1:1 + n_out] = dy
    y, z = ops.linear_fwd(x, w, b, act="silu", residual=r, train=True)
    y2, z2 = ops.linear_fwd(wide[:, 3:3 + n_in], w, b, act="silu", residual=r, train=True)
    assert torch.equal(y, y2) and torch.equal(z, z2)
    g = ops.linear_bwd(dy, x, w, z, act="silu")
    g2 = ops.linear_bwd(dwide[:, 1:1 + n_out], wide[:, 3:3 + n_in], w, z, act="silu")
    assert all(torch.equal(p, q) for p, q in zip(g, g2))
    assert float(wide[:, :3].abs().max()) == 0.0 and float(wide[:, 3 + n_in:].abs().max()) == 0.0
    bad = x.clone()
    bad[rows - 1, 7] = float("inf")
    dx, dw, db = ops.linear_bwd(dy, bad, w, z, act="silu")
    assert torch.equal(dx, g[0]) and torch.equal(db, g[2])
    keep = [c for c in range(n_in) if c != 7]
    assert torch.equal(dw[:, keep], g[1][:, keep]) and not bool(torch.isfinite(dw[:, 7]).any())


@pytest.mark.gpu
def test_linear_heads_in_a_graph():
    """replayed with other inputs and eager work in between, against the eager calls, bit for bit"""
    from fneus import ops
    x, w, b, r, dy = inputs(5000, 300, 3, torch.float32)

    def run():
        y, z = ops.linear_fwd(x, w, b, act="softplus", residual=r, train=True)
        return (y,) + ops.linear_bwd(dy, x, w, z, act="softplus")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        for t, s in zip((x, w, b, r, dy), inputs(5000, 300, 3, torch.float32, seed=k + 1)):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, run()))


# More workgroups than 2^32 threads hold, which is what a launch takes along its first dimension
@pytest.mark.gpu
@pytest.mark.parametrize("rows,n_in,n_out", [((1 << 27) + 37, 264, 2), ((1 << 30) + 70, 8, 1)], ids=["head", "tiled"])
def test_linear_more_rows_than_a_launch_takes(rows, n_in, n_out):
    """heads of 2^27 rows (512 threads per 16 of them), few outputs of 2^30 rows (256 threads per 64): forward, and the tiled input gradient.  All
    rows but the last hundred are one row seen again: the same bits in every place (a row's sums do not depend on its place)"""
    from fneus import ops
    g = torch.Generator().manual_seed(6)
    near = torch.randn(100, n_in, generator=g).bfloat16().cuda()
    w = (torch.randn(n_out, n_in, generator=g) / math.sqrt(n_in)).bfloat16().cuda()
    x = torch.empty(rows, n_in, dtype=torch.bfloat16, device="cuda")
    x[:-100] = near[:1]
    x[-100:] = near
    y = ops.linear_fwd(x, w, act="silu")[0]
    zd = near.double() @ w.double().t()
    want = act64(zd, "silu")
    lim = (1.13 * sums(n_in) + 4 * 2.0 ** -23) * (near.double().abs() @ w.double().abs().t()) + half(torch.bfloat16) * want.abs()
    check(y[-100:], want, lim + torch.finfo(torch.bfloat16).smallest_normal, "y")
    check(y[:1], want[:1], lim[:1] + torch.finfo(torch.bfloat16).smallest_normal, "y")
    same = y[0].clone()
    assert bool((y[:-100] == same).all())
    if n_in == 8:
        del y
        dy = torch.empty(rows, n_out, dtype=torch.bfloat16, device="cuda")
        dy[:-100], dy[-100:] = 0.5, near[:, :n_out]
        dx = ops.linear_bwd(dy, x, w, need=(True, False, False))[0]
        want = near[:, :n_out].double() @ w.double()
        check(dx[-100:], want, (half(torch.bfloat16) + sums(n_out)) * want.abs() + torch.finfo(torch.bfloat16).smallest_normal, "dx")
        assert bool((dx[:-100] == (0.5 * w.float()).bfloat16()[0]).all())


@pytest.mark.gpu
def test_linear_gelu_keeps_its_digits_in_the_tail():
    """fp32 GELU and its derivative relative to their own size, through identity weights (z = x and dx = delta to the last bit: three bf16 terms hold 24).
    exp(-z^2 / 2): the argument is off by six roundings (1 / sqrt 2, the product, the square twice over, log2 e, the product) of z^2 / 2 each, 3 z^2 2^-24;
    the instructions' ulp, nine steps of the polynomial and four products: at most 16 + 8 x 2^-24 more"""
    from fneus import ops
    z = torch.linspace(-8.0, 8.0, 4096 * 64, device="cuda").reshape(-1, 64).contiguous()
    eye = torch.eye(64, device="cuda")
    for rows in (8, 500, 4096):                     # (each form of the product)
        x = z[:: 4096 // rows].contiguous()
        y, zz = ops.linear_fwd(x, eye, act="gelu", train=True)
        assert torch.equal(zz, x)
        d = x.double()
        want = act64(d, "gelu")
        rel = (3 * d * d + 24) * 2.0 ** -24
        check(y, want, rel * want.abs(), "gelu")
        dx = ops.linear_bwd(torch.ones_like(x), x, eye, zz, act="gelu", need=(True, False, False))[0]
        pdf = torch.exp(-d * d / 2) / math.sqrt(2 * math.pi)
        check(dx, dact64(d, "gelu"), rel * (0.5 * torch.special.erfc(-d * math.sqrt(0.5)) + d.abs() * pdf), "gelu'")


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["sigmoid", "softplus", "gelu", "silu"])
def test_linear_gradient_at_pre_activations_beyond_fp16(act):
    """z = -160000 and +160000 in fp16 rows: stored as infinities; the derivative there is its limit (0, and 1 or 0), not NaN; a NaN stays one"""
    from fneus import ops
    for rows, n_out in ((4, 24), (500, 24), (9000, 24), (9000, 3)):        # (each form)
        x = torch.full((rows, 8), 200.0, dtype=torch.float16, device="cuda")
        x[1] = -200.0
        x[2, 0] = float("nan")
        w = torch.full((n_out, 8), -100.0, dtype=torch.float16, device="cuda")
        y, z = ops.linear_fwd(x, w, act=act, train=True)
        assert bool(torch.isinf(z[0]).all()) and bool(torch.isfinite(y[0]).all()) and bool((y[0] == 0).all())
        dy = torch.full((rows, n_out), 2.0 ** -7, dtype=torch.float16, device="cuda")
        dx, dw, db = ops.linear_bwd(dy, x, w, z, act=act)
        assert bool((dx[0] == 0).all()) and bool((dx[3:] == 0).all()) and bool(torch.isnan(dx[2]).all())
        up = 0.0 if act == "sigmoid" else -100.0 * n_out * 2.0 ** -7
        assert bool((dx[1] == up).all()), (rows, n_out, dx[1])
        clean = [k for k in range(rows) if k != 2]
        db = ops.linear_bwd(dy[clean], x[clean], w, z[clean], act=act)[2]
        assert bool((db == (0.0 if act == "sigmoid" else 2.0 ** -7)).all())
