"""Layer norm, forward and backward, against its formulas in 64 bits.

Tolerances.  u = 2^-24 is half a step of f32.  A sum of n terms in any order is off by at most n u sum|t|; with the
kernels' orders (serial runs of at most n / 32 + 16 terms) `depth` = n / 32 + 32 covers it and the few operations on
each term.  mean: depth u mean|x|.  rstd: relative (depth + 4) u, plus the mean's own error, which enters squared.  y:
the error of x - mean (the mean's and one rounding) times |rstd gamma|, plus relative ones of y - beta, plus one
rounding of y.  dgamma and dbeta: rows u sum|dy xhat| for any order, and xhat's own error.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = [(1, 1), (1, 2), (3, 5), (1, 4096), (7, 31), (64, 32), (33, 128), (5, 129), (300, 256), (257, 100),
         (1000, 512), (19, 1000), (40, 1024), (9, 1111), (13, 2048), (600, 2052), (3, 4100), (4, 8192), (2, 8193),
         (3, 16384), (2, 20001), (1, 70000)]


def _forward64(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    y = (x - mean) * rstd
    if gamma is not None:
        y = y * gamma.double()
    if beta is not None:
        y = y + beta.double()
    return y, mean, rstd


def _tolerances(x, gamma, y, beta, mean, rstd):
    n = x.shape[1]
    depth = n / 32 + 32
    dm = depth * U * x.double().abs().mean(1, keepdim=True)
    dr = (depth + 4) * U + (dm * rstd) ** 2
    g = gamma.double().abs() if gamma is not None else 1.0
    core = (y - (beta.double() if beta is not None else 0)).abs()
    dy = (dm + U * (x.double() - mean).abs()) * rstd * g + core * (dr + 3 * U) + 2 * U * y.abs()
    return dy + 1e-30, dm + 1e-30, dr * rstd


def _make(dev, rows, cols, pad, shift, seed, offset=3.0):
    t = dev.torch
    g = t.Generator(device="cuda").manual_seed(seed)
    buf = t.randn(rows * (cols + pad) + shift, generator=g, device="cuda") * 2 + offset
    x = buf[shift:].view(rows, cols + pad)[:, :cols]
    return x, 1 + 0.2 * t.randn(cols, generator=g, device="cuda"), t.randn(cols, generator=g, device="cuda")


def _ptr(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("pad,shift,affine", [(0, 0, "both"), (3, 1, "both"), (4, 0, "gamma"), (0, 0, "beta"),
                                              (0, 4, "none")])
def test_forward(jx, dev, rows, cols, pad, shift, affine):
    t = dev.torch
    x, gamma, beta = _make(dev, rows, cols, pad, shift, rows * 7 + cols)
    gamma = gamma if affine in ("both", "gamma") else None
    beta = beta if affine in ("both", "beta") else None
    y = t.full((rows, cols + pad), 7.0, device="cuda")
    mean, rstd = t.full((rows,), np.nan, device="cuda"), t.full((rows,), np.nan, device="cuda")
    jx.layernorm(x.data_ptr(), _ptr(gamma), _ptr(beta), y.data_ptr(), rows, cols, 1e-5, mean.data_ptr(),
                 rstd.data_ptr(), x.stride(0), cols + pad, dev.stream)
    wy, wm, wr = _forward64(x, gamma, beta, 1e-5)
    ty, tm, tr = _tolerances(x, gamma, wy, beta, wm, wr)
    assert bool(((y[:, :cols].double() - wy).abs() <= ty).all())
    assert bool(((mean.double()[:, None] - wm).abs() <= tm).all())
    assert bool(((rstd.double()[:, None] - wr).abs() <= tr).all())
    assert bool((y[:, cols:] == 7.0).all())  # the rows' padding is left as it was


def test_forward_in_place_and_without_statistics(jx, dev):
    x, gamma, beta = _make(dev, 37, 515, 1, 0, 5)
    y = dev.empty((37, 515))
    jx.layernorm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), 37, 515, ldx=x.stride(0),
                 stream=dev.stream)
    jx.layernorm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), x.data_ptr(), 37, 515, ldx=x.stride(0),
                 ldy=x.stride(0), stream=dev.stream)
    assert bool((x == y).all())


def test_forward_far_from_zero(jx, dev):
    """A mean 1000 times the spread: the variance is of the centred values, not a difference of large squares."""
    x, gamma, beta = _make(dev, 50, 1000, 0, 0, 6, offset=2000.0)
    y, mean, rstd = dev.empty((50, 1000)), dev.empty((50,)), dev.empty((50,))
    jx.layernorm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), 50, 1000, 1e-5, mean.data_ptr(),
                 rstd.data_ptr(), stream=dev.stream)
    wy, wm, wr = _forward64(x, gamma, beta, 1e-5)
    ty, tm, tr = _tolerances(x, gamma, wy, beta, wm, wr)
    assert bool(((y.double() - wy).abs() <= ty).all())
    assert bool(((rstd.double()[:, None] - wr).abs() <= tr).all())


def test_non_finite_rows_stay_apart(jx, dev):
    t = dev.torch
    x, gamma, beta = _make(dev, 6, 300, 0, 0, 8)
    clean = dev.empty((6, 300))
    jx.layernorm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), clean.data_ptr(), 6, 300, stream=dev.stream)
    x[2, 17] = float("nan")
    x[4, 299] = float("inf")
    y = dev.empty((6, 300))
    jx.layernorm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), 6, 300, stream=dev.stream)
    good = [0, 1, 3, 5]
    assert bool((y[good] == clean[good]).all())
    assert bool(t.isnan(y[[2, 4]]).all())


@pytest.mark.parametrize("rows,cols", SIZES + [(5000, 64), (2500, 333), (300, 8500), (250, 16384), (400, 9001)])
@pytest.mark.parametrize("pad,shift,affine,wanted", [(0, 0, True, "all"), (3, 1, True, "all"), (4, 0, False, "all"),
                                                     (0, 0, True, "dx"), (0, 0, True, "weights"),
                                                     (0, 0, True, "gamma"), (0, 0, True, "beta")])
def test_backward(jx, dev, rows, cols, pad, shift, affine, wanted):
    t = dev.torch
    x, gamma, _ = _make(dev, rows, cols, pad, shift, rows + cols)
    dy, _, _ = _make(dev, rows, cols, pad, shift, rows + cols + 1, offset=0.25)
    gamma = gamma if affine else None
    _, mean, rstd = (v.float().reshape(-1) if i else v for i, v in enumerate(_forward64(x, None, None, 1e-5)))
    dx = t.full((rows, cols + pad), 7.0, device="cuda") if wanted in ("all", "dx") else None
    dg = t.full((cols,), np.nan, device="cuda") if wanted in ("all", "weights", "gamma") else None
    db = t.full((cols,), np.nan, device="cuda") if wanted in ("all", "weights", "beta") else None
    jx.layernorm_bwd(dy.data_ptr(), x.data_ptr(), _ptr(gamma), mean.data_ptr(), rstd.data_ptr(), _ptr(dx), _ptr(dg),
                     _ptr(db), rows, cols, dy.stride(0), x.stride(0), cols + pad, dev.stream)
    xd, d, m, r = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    xhat = (xd - m) * r
    # xhat's own error: the difference is rounded once, the product once
    g = d * (gamma.double() if affine else 1.0)
    c1, c2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    depth = cols / 32 + 32
    if dx is not None:
        want = (g - c1 - xhat * c2) * r
        tol = U * r * (4 * g.abs() + (depth + 4) * g.abs().mean(1, keepdim=True) + 8 * (xhat * c2).abs()
                       + xhat.abs() * (depth + 8) * (g * xhat).abs().mean(1, keepdim=True)) + 1e-30
        assert bool(((dx[:, :cols].double() - want).abs() <= tol).all())
        assert bool((dx[:, cols:] == 7.0).all())
    if dg is not None:
        assert bool(((dg.double() - (d * xhat).sum(0)).abs() <= (rows + 4) * U * (d * xhat).abs().sum(0)).all())
    if db is not None:
        assert bool(((db.double() - d.sum(0)).abs() <= (rows + 1) * U * d.abs().sum(0)).all())


def test_backward_in_place_and_repeatable(jx, dev):
    x, gamma, _ = _make(dev, 700, 260, 0, 0, 2)
    dy, _, _ = _make(dev, 700, 260, 0, 0, 3)
    _, mean, rstd = (v.float().reshape(-1) if i else v for i, v in enumerate(_forward64(x, None, None, 1e-5)))
    outs = []
    for k in range(3):
        src = dy.clone()
        dx = src if k == 2 else dev.empty((700, 260))
        dg, db = dev.empty((260,)), dev.empty((260,))
        jx.layernorm_bwd(src.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                         dx.data_ptr(), dg.data_ptr(), db.data_ptr(), 700, 260, stream=dev.stream)
        outs.append((dx, dg, db))
    for other in outs[1:]:
        assert all(bool((a == b).all()) for a, b in zip(outs[0], other))


def test_backward_no_rows(jx, dev):
    dg, db = dev.full((9,), 3.0), dev.full((9,), 3.0)
    jx.layernorm_bwd(None, None, None, None, None, None, dg.data_ptr(), db.data_ptr(), 0, 9, stream=dev.stream)
    assert float(dg.abs().sum()) == 0.0 and float(db.abs().sum()) == 0.0


def test_backward_against_differences(jx, dev):
    """The directional derivative of sum(dy * y) by central differences of the formula in 64 bits.  The step h = 1e-5
    leaves an error of h^2 (about 1e-10 relative); the kernel's is the sums' n u, here below 1e-4 of the parts."""
    t = dev.torch
    rows, cols = 23, 77
    x, gamma, beta = _make(dev, rows, cols, 0, 0, 4)
    dy, _, _ = _make(dev, rows, cols, 0, 0, 9, offset=0.0)
    y, mean, rstd = dev.empty((rows, cols)), dev.empty((rows,)), dev.empty((rows,))
    jx.layernorm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), rows, cols, 1e-5, mean.data_ptr(),
                 rstd.data_ptr(), stream=dev.stream)
    dx, dg, db = dev.empty((rows, cols)), dev.empty((cols,)), dev.empty((cols,))
    jx.layernorm_bwd(dy.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
                     dg.data_ptr(), db.data_ptr(), rows, cols, stream=dev.stream)
    g = t.Generator(device="cuda").manual_seed(1)
    for value, grad in ((x, dx), (gamma, dg), (beta, db)):
        e = t.randn(value.shape, generator=g, device="cuda", dtype=t.float64)

        def loss(h):
            args = [v.double() + (h * e if v is value else 0) for v in (x, gamma, beta)]
            return float((_forward64(*args, 1e-5)[0] * dy.double()).sum())

        want = (loss(1e-5) - loss(-1e-5)) / 2e-5
        parts = float((grad.double() * e).abs().sum())
        assert abs(float((grad.double() * e).sum()) - want) <= 1e-4 * parts


def test_captured_and_replayed(jx, dev):
    t = dev.torch
    x, gamma, beta = _make(dev, 130, 384, 0, 0, 11)
    dy = t.randn(130, 384, device="cuda")
    y, mean, rstd = dev.empty((130, 384)), dev.empty((130,)), dev.empty((130,))
    dx, dg, db = dev.empty((130, 384)), dev.empty((384,)), dev.empty((384,))

    def step():
        st = dev.stream
        jx.layernorm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), 130, 384, 1e-5, mean.data_ptr(),
                     rstd.data_ptr(), stream=st)
        jx.layernorm_bwd(dy.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                         dx.data_ptr(), dg.data_ptr(), db.data_ptr(), 130, 384, stream=st)

    step()
    dev.sync()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        step()
    x.add_(t.randn_like(x))
    step()
    dev.sync()
    want = [v.clone() for v in (y, dx, dg, db)]
    for v in (y, dx, dg, db):
        v.zero_()
    graph.replay()
    dev.sync()
    assert all(bool((a == b).all()) for a, b in zip(want, (y, dx, dg, db)))
