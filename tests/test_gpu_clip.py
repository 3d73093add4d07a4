"""The global gradient norm and clipping against 64 bits.

Tolerances: squares and sums are in f64, so the norm is the f64 value rounded to f32 (2^-24 relative, doubled for the
square root's and the sum's own last places in f64); an output is g times a factor rounded to f32, rounded again:
2 * 2^-24, and 2^-24 more for the norm's own error in f64, far below that.
"""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _tables(ts):
    return (C.c_void_p * max(1, len(ts)))(*[t.data_ptr() if t.numel() else None for t in ts])


def _sizes(ts):
    return (C.c_int64 * max(1, len(ts)))(*[t.numel() for t in ts])


def _tensors(dev, sizes, seed, shift=0):
    g = dev.torch.Generator(device="cuda").manual_seed(seed)
    flat = dev.torch.randn(sum(sizes) + shift, generator=g, device="cuda")
    out, at = [], shift
    for n in sizes:
        out.append(flat[at:at + n])
        at += n
    return out


def _norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


LISTS = [[1], [0, 5, 0], [3, 1, 4, 1, 5, 9, 2, 6], [8192], [8191, 8193, 1], [100003], [4096] * 130, [7] * 700,
         [1 << 20, 1, 1 << 18, 333], [5_000_001]]


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("ratio", [0.25, 4.0])
def test_norm_and_clip(jx, dev, sizes, shift, ratio):
    gs = _tensors(dev, sizes, len(sizes) + max(sizes), shift)
    outs = [dev.full((n,), np.nan) for n in sizes]
    norm, norm2 = dev.full((1,), np.nan), dev.full((1,), np.nan)
    want = _norm64(gs)
    limit = want * ratio
    jx.grad_norm(_tables(gs), _sizes(gs), len(gs), norm.data_ptr(), dev.stream)
    jx.clip_grads(_tables(gs), _tables(outs), _sizes(gs), len(gs), limit, norm2.data_ptr(), dev.stream)
    assert abs(float(norm) - want) <= 2 * U * want
    assert float(norm) == float(norm2)
    factor = min(1.0, limit / (want + 1e-6))
    for g, o in zip(gs, outs):
        if ratio > 1:
            assert bool((o == g).all())
        else:
            assert bool(((o.double() - g.double() * factor).abs() <= 3 * U * (g.double() * factor).abs()).all())
    # in place: the same values
    jx.clip_grads(_tables(gs), _tables(gs), _sizes(gs), len(gs), limit, None, dev.stream)
    assert all(bool((g == o).all()) for g, o in zip(gs, outs))


def test_no_tensors(jx, dev):
    norm = dev.full((1,), np.nan)
    jx.grad_norm(None, None, 0, norm.data_ptr(), dev.stream)
    assert float(norm) == 0.0
    jx.clip_grads(None, None, None, 0, 1.0, norm.data_ptr(), dev.stream)
    assert float(norm) == 0.0


def test_large_and_tiny_values(jx, dev):
    """Squares beyond f32's range at both ends."""
    for v in (1e30, 1e-30):
        g = dev.full((1000,), v)
        norm = dev.full((1,), np.nan)
        jx.grad_norm(_tables([g]), _sizes([g]), 1, norm.data_ptr(), dev.stream)
        want = float(g.double().square().sum().sqrt())
        assert abs(float(norm) - want) <= 2 * U * want


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite(jx, dev, bad):
    t = dev.torch
    g = t.ones(5000, device="cuda")
    g[4321] = bad
    o, norm = dev.empty((5000,)), dev.empty((1,))
    jx.clip_grads(_tables([g]), _tables([o]), _sizes([g]), 1, 1.0, norm.data_ptr(), dev.stream)
    if math.isnan(bad):
        assert bool(t.isnan(norm).all()) and bool(t.isnan(o).all())
    else:
        assert float(norm) == math.inf
        assert bool(t.isnan(o[4321])) and float(o[:4321].abs().sum()) == 0.0


def test_repeatable(jx, dev):
    gs = _tensors(dev, [30011, 17, 250000], 3)
    seen = set()
    for _ in range(5):
        norm = dev.empty((1,))
        jx.grad_norm(_tables(gs), _sizes(gs), 3, norm.data_ptr(), dev.stream)
        seen.add(float(norm))
    assert len(seen) == 1


def test_clip_then_adam(jx, dev, oracle):
    """As a training step uses them: clipped in place, then jx_adam_step_f32, against the same step in the oracle."""
    rng = np.random.default_rng(4)
    sizes = [513, 64]
    ps = [rng.standard_normal(n).astype(np.float32) for n in sizes]
    gs = [rng.standard_normal(n).astype(np.float32) * 10 for n in sizes]
    P, G = [dev.put(p) for p in ps], [dev.put(g) for g in gs]
    M, V = [dev.full((n,), 0.0) for n in sizes], [dev.full((n,), 0.0) for n in sizes]
    jx.clip_grads(_tables(G), _tables(G), _sizes(G), 2, 1.0, None, dev.stream)
    jx.call("jx_adam_step_f32", _tables(P), _tables(G), _tables(M), _tables(V), _sizes(G), 2, 1e-3, 0.9, 0.999, 1e-8,
            1, dev.stream)
    for i in range(2):
        clipped = dev.get(G[i])
        want, _, _ = oracle.adam_update(ps[i], clipped, np.zeros_like(ps[i]), np.zeros_like(ps[i]), 1e-3, 0.9, 0.999,
                                        1e-8, 1, True)
        assert np.array_equal(dev.get(P[i]), want)
    total = math.sqrt(sum(float((dev.get(g).astype(np.float64) ** 2).sum()) for g in G))
    assert abs(total - 1.0) <= 1e-5  # the factor's 1e-6 in its denominator and the roundings


def test_captured_and_replayed(jx, dev):
    t = dev.torch
    gs = _tensors(dev, [1000, 70001], 12)
    outs = [dev.full((g.numel(),), 0.0) for g in gs]
    norm = dev.empty((1,))
    a, b, n = _tables(gs), _tables(outs), _sizes(gs)
    jx.clip_grads(a, b, n, 2, 1.0, norm.data_ptr(), dev.stream)
    dev.sync()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        jx.clip_grads(a, b, n, 2, 1.0, norm.data_ptr(), dev.stream)
    for g in gs:
        g.mul_(3.0)
    graph.replay()
    dev.sync()
    want = _norm64(gs)
    assert abs(float(norm) - want) <= 2 * U * want
    for g, o in zip(gs, outs):
        f = 1.0 / (want + 1e-6)
        assert bool(((o.double() - g.double() * f).abs() <= 3 * U * (g.double() * f).abs()).all())
