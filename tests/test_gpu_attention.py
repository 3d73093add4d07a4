"""Attention over packed sequences, forward and backward, against its formulas in 64 bits.

Tolerances.  With A[i] = max over visible j of scale * sum_e |q[i,e] k[j,e]|, a score is off by at most
delta[i] = A[i] * (2^-21 + (dim + 32) 2^-24): both operands are held to 22 bits, the sum has dim terms.  A weight is off
by that relatively, the exponential and the sums' own roundings add (32 + sqrt(keys)) 2^-24, and the normalisation
doubles it: |o - want| <= 2 (delta + (64 + sqrt(keys)) 2^-24 + 2^-21) sum_j p |v|.  Norms over all outputs, where roundings
average out, are held to the library's bound for products, 1e-5.
Gradients: dout v^T and rowsum(dout o) are each off by at most about 2^-20 of the sum of their terms' magnitudes, so
ds = p (dp - delta) by that share of p (|dout| |v| + |dout| |o|); `mag` is that magnitude taken on to the output.
||error|| <= 2e-6 ||mag|| + 1e-5 ||want||, the second term for p's own error.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Case:
    """Inputs, outputs with the value 7 in them, and the call."""

    def __init__(self, dev, q_lens, k_lens, heads, kv_heads, dim, causal=True, pad=0, tail=0, head=0, shift=0, seed=0,
                 spread=1.5):
        t = self.t = dev.torch
        self.dev, self.heads, self.kv_heads, self.dim, self.causal = dev, heads, kv_heads, dim, causal
        self.q_lens, self.k_lens = q_lens, k_lens
        self.cq = list(np.cumsum([head] + q_lens))
        self.ck = list(np.cumsum([head] + k_lens))
        self.tq, self.tk = self.cq[-1] + tail, self.ck[-1] + tail
        self.scale = dim ** -0.5
        self.gen = t.Generator(device="cuda").manual_seed(seed + sum(q_lens) + 31 * dim)
        self.pad, self.shift = pad, shift
        self.q = self.buf(self.tq, heads).mul_(spread)
        self.k, self.v = self.buf(self.tk, kv_heads), self.buf(self.tk, kv_heads)
        self.dout = self.buf(self.tq, heads)
        self.o = self.buf(self.tq, heads, 7.0)
        self.lse = t.full((heads, self.tq), 7.0, device="cuda")
        self.dq, self.dk, self.dv = self.buf(self.tq, heads, 7.0), self.buf(self.tk, kv_heads, 7.0), self.buf(
            self.tk, kv_heads, 7.0)
        self.cu_q = t.tensor(self.cq, dtype=t.int32, device="cuda")
        self.cu_k = t.tensor(self.ck, dtype=t.int32, device="cuda")

    def buf(self, rows, heads, fill=None):
        t, row = self.t, heads * self.dim + self.pad
        flat = t.empty(rows * row + self.shift + 1, device="cuda")
        if fill is None:
            flat.normal_(generator=self.gen)
        else:
            flat.fill_(fill)
        return flat[self.shift:self.shift + rows * row].view(rows, row)[:, :heads * self.dim].unflatten(
            1, (heads, self.dim))

    def sizes(self, **more):
        ld = lambda x: x.stride(0) if x.shape[0] else x.shape[1] * self.dim + self.pad
        return {**dict(batch=len(self.q_lens), total_q=self.tq, total_k=self.tk, heads=self.heads,
                       kv_heads=self.kv_heads, head_dim=self.dim, max_q=max(self.q_lens, default=0),
                       max_k=max(self.k_lens, default=0), ldq=ld(self.q), ldk=ld(self.k), ldv=ld(self.v),
                       ldo=ld(self.o), scale=self.scale, causal=self.causal, stream=self.dev.stream), **more}

    def forward(self, jx, **more):
        jx.attention(self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.o.data_ptr(), self.lse.data_ptr(),
                     self.cu_q.data_ptr(), self.cu_k.data_ptr(), **self.sizes(**more))

    def backward(self, jx, **more):
        jx.attention_bwd(self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.o.data_ptr(),
                         self.lse.data_ptr(), self.dout.data_ptr(), self.dq.data_ptr(), self.dk.data_ptr(),
                         self.dv.data_ptr(), self.cu_q.data_ptr(), self.cu_k.data_ptr(), **self.sizes(**more))

    def reference(self, grads=False):
        """o, lse and o's bound; with grads also dq, dk, dv and their magnitudes; 7 in rows of no sequence."""
        t = self.t
        f = lambda x: t.full(x.shape, 7.0, dtype=t.float64, device="cuda")
        o, lse, bound = f(self.o), f(self.lse), t.zeros(self.o.shape, dtype=t.float64, device="cuda")
        g = [f(self.dq), f(self.dk), f(self.dv)]
        m = [t.zeros(x.shape, dtype=t.float64, device="cuda") for x in g]
        for a, b, c, d in zip(self.cq, self.cq[1:], self.ck, self.ck[1:]):
            for x in g[1:]:
                x[c:d] = 0
            i, j = t.arange(b - a, device="cuda")[:, None], t.arange(d - c, device="cuda")[None]
            seen = (j <= i + (d - c) - (b - a)) if self.causal else (j >= 0) & (i >= 0)
            for h in range(self.heads):
                hk = h // (self.heads // self.kv_heads)
                q, k, v = self.q[a:b, h].double(), self.k[c:d, hk].double(), self.v[c:d, hk].double()
                x = (q @ k.t() * self.scale).masked_fill(~seen, -math.inf)
                z = t.logsumexp(x, 1) if d > c else t.full((b - a,), -math.inf, dtype=t.float64, device="cuda")
                p = (x - z.masked_fill(z == -math.inf, 0.0)[:, None]).exp()
                # keys that a row does not see take no part in it, whatever they hold
                vz = v.nan_to_num(0.0, 0.0, 0.0)
                o[a:b, h], lse[h, a:b] = p @ vz, z
                if d > c:
                    mag = (q.abs() @ k.abs().t() * self.scale).masked_fill(~seen, 0.0).amax(1, keepdim=True)
                    u = 2.0 ** -24
                    eps = mag * (8 * u + (self.dim + 32) * u) + (64 + math.sqrt(d - c)) * u + 8 * u
                    bound[a:b, h] = 2 * eps * (p @ vz.abs()) + 1e-30
                if grads:
                    do = self.dout[a:b, h].double()
                    dp = do @ v.t()
                    ds = p * (dp - (do * o[a:b, h]).sum(1, keepdim=True)) * self.scale
                    dsm = p * (do.abs() @ v.abs().t() + (do * o[a:b, h]).abs().sum(1, keepdim=True)) * self.scale
                    g[0][a:b, h], m[0][a:b, h] = ds @ k, dsm @ k.abs()
                    g[1][c:d, hk] += ds.t() @ q
                    m[1][c:d, hk] += dsm.t() @ q.abs()
                    g[2][c:d, hk] += p.t() @ do
                    m[2][c:d, hk] += p.t() @ do.abs()
        return (o, lse, bound, g, m) if grads else (o, lse, bound)

    def check_forward(self):
        o, lse, bound = self.reference()
        d = (self.o.double() - o).abs()
        assert bool((d <= bound).all()), float((d / (bound + 1e-300)).max())
        assert float(d.norm()) <= 1e-5 * float(o.norm()) + 1e-30
        assert bool((self.t.isinf(lse) == self.t.isinf(self.lse)).all())
        e = (self.lse.double() - lse).masked_fill(self.t.isinf(lse), 0.0).abs()
        assert bool((e <= 1e-5 * (1 + lse.masked_fill(self.t.isinf(lse), 0.0).abs())).all())

    def check_backward(self):
        _, _, _, g, m = self.reference(True)
        for name, got, want, mag in zip(("dq", "dk", "dv"), (self.dq, self.dk, self.dv), g, m):
            off = float((got.double() - want).norm())
            assert off <= 2e-6 * float(mag.norm()) + 1e-5 * float(want.norm()), (name, off, float(want.norm()))


# q_lens, k_lens, heads, kv_heads, dim, causal
FORWARD = [
    ([1], [1], 1, 1, 128, True), ([1], [1], 2, 1, 1, True), ([7], [7], 3, 3, 5, True), ([128], [128], 2, 2, 64, True),
    ([127], [127], 2, 1, 128, True), ([129], [129], 2, 1, 128, True), ([256], [256], 1, 1, 128, False),
    ([300], [300], 4, 2, 127, True), ([64, 1, 0, 200, 33], [64, 1, 0, 200, 33], 4, 4, 80, True),
    ([5, 0, 3], [0, 9, 2], 2, 1, 64, True), ([5, 0, 3], [0, 9, 2], 2, 1, 64, False), ([200], [50], 2, 2, 64, True),
    ([300, 10], [140, 500], 6, 2, 128, True), ([513], [1025], 2, 1, 64, False), ([1000], [1000], 3, 1, 96, True),
    ([1] * 9, [1, 2, 130, 1000, 64, 3, 0, 257, 4096], 8, 2, 128, True), ([1] * 5, [700, 3, 0, 1, 65], 8, 8, 64, True),
    ([2, 4, 1], [3000, 100, 5], 4, 4, 128, True), ([1, 1], [2049, 77], 16, 1, 40, False), ([3], [20000], 12, 4, 72, True),
    ([1], [33000], 16, 1, 128, True), ([1] * 200, [17] * 200, 2, 1, 32, True), ([30] * 40, [30] * 40, 2, 1, 64, True),
    ([2000], [2000], 2, 1, 128, True), ([16], [16], 5, 1, 128, True), ([17], [900], 8, 1, 128, True),
]
LAYOUTS = [dict(), dict(pad=4, tail=3), dict(pad=3, shift=1, head=2, tail=1)]


def _id(v):
    return "x".join(map(str, v[:4])) + f"n{len(v)}" if isinstance(v, list) else None


@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim,causal", FORWARD, ids=_id)
@pytest.mark.parametrize("layout", LAYOUTS, ids=["dense", "strided", "shifted"])
def test_forward(jx, dev, q_lens, k_lens, heads, kv_heads, dim, causal, layout):
    c = Case(dev, q_lens, k_lens, heads, kv_heads, dim, causal, **layout)
    c.forward(jx)
    c.check_forward()
    assert jx.device_status() == 0


@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim,causal", FORWARD, ids=_id)
@pytest.mark.parametrize("layout", LAYOUTS, ids=["dense", "strided", "shifted"])
def test_backward(jx, dev, q_lens, k_lens, heads, kv_heads, dim, causal, layout):
    c = Case(dev, q_lens, k_lens, heads, kv_heads, dim, causal, **layout)
    c.forward(jx)
    c.backward(jx)
    c.check_backward()
    assert jx.device_status() == 0


@pytest.mark.parametrize("hint", [(0, 0), (1, 1), (1, 100000), (5000, 5000)])
def test_any_hint_gives_the_result(jx, dev, hint):
    c = Case(dev, [150, 1, 20], [150, 700, 20], 4, 2, 64)
    c.forward(jx, max_q=hint[0], max_k=hint[1])
    c.check_forward()
    c.backward(jx, max_q=hint[0], max_k=hint[1])
    c.check_backward()


def test_without_lse(jx, dev):
    c = Case(dev, [40, 260], [40, 260], 4, 2, 64)
    c.forward(jx)
    want = c.o.clone()
    c.o.fill_(7.0)
    jx.attention(c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.o.data_ptr(), None, c.cu_q.data_ptr(),
                 c.cu_k.data_ptr(), **c.sizes())
    assert bool((want == c.o).all())


@pytest.mark.parametrize("q_lens,k_lens", [([200], [200]), ([1, 1], [500, 3]), ([40, 40], [40, 300])])
def test_values_of_unseen_keys_do_not_matter(jx, dev, q_lens, k_lens):
    """NaN and infinities behind a row's last visible key, and in rows of no sequence."""
    c = Case(dev, q_lens, k_lens, 4, 2, 64, tail=5, head=3)
    for x in (c.k, c.v):
        x[:3], x[-5:] = float("nan"), float("inf")
    c.q[:3], c.q[-5:] = float("nan"), float("inf")
    c.forward(jx)
    c.check_forward()
    # the last key of the first sequence is seen by its last row alone
    last, row = c.ck[1] - 1, c.cq[1] - 1
    before = c.o.clone()
    c.k[last], c.v[last] = float("nan"), float("inf")
    c.forward(jx)
    keep = [r for r in range(c.tq) if r != row]
    assert float((c.o[keep] - before[keep]).abs().max()) <= 1e-5
    assert bool(c.t.isnan(c.o[row]).all())


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e18])
def test_values_of_any_size(jx, dev, size):
    """v scales the outputs; q and k scale against one another."""
    c = Case(dev, [140, 1], [140, 300], 2, 1, 64)
    c.v.mul_(size)
    c.q.mul_(size)
    c.k.div_(size)
    c.forward(jx)
    o, _, bound = c.reference()
    assert bool(((c.o.double() - o).abs() <= bound).all())


def test_rows_of_very_different_sizes(jx, dev):
    """One key and one value 2^30 times the others: the small ones keep their own precision."""
    c = Case(dev, [200], [200], 2, 1, 64, spread=0.1)
    big = 2.0 ** 30
    c.k[150] = -c.q[:, 0].sign()[150] * big  # far below every score that matters, or far above
    c.v[150] *= big
    c.forward(jx)
    o, _, bound = c.reference()
    assert bool(((c.o.double() - o).abs() <= bound).all())


def test_scores_far_apart(jx, dev):
    """Weights that underflow, and a first block of keys far below the later ones."""
    c = Case(dev, [300], [300], 2, 2, 64, spread=40.0)
    c.k[:128].mul_(0.01)
    c.forward(jx)
    c.check_forward()
    c.backward(jx)
    c.check_backward()


def test_gradients_against_differences(jx, dev):
    """The directional derivative of sum(dout * o), by central differences of the formula in 64 bits.  The step of 1e-4
    leaves about 1e-8 relative; the kernel's own error stays below 1e-4 of the parts' magnitudes."""
    c = Case(dev, [50, 170], [60, 130], 4, 2, 32)
    c.forward(jx)
    c.backward(jx)
    t = c.t
    for name in ("q", "k", "v"):
        value, grad = getattr(c, name), getattr(c, "d" + name)
        e = t.randn(value.shape, generator=c.gen, device="cuda", dtype=t.float64)

        def loss(h):
            setattr(c, name, value.double() + h * e)
            return float((c.reference()[0] * c.dout.double()).sum())

        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        setattr(c, name, value)
        parts = float((grad.double() * e).abs().sum())
        assert abs(float((grad.double() * e).sum()) - want) <= 1e-4 * parts


def test_repeatable(jx, dev):
    c = Case(dev, [700, 90], [700, 400], 8, 2, 128)
    runs = []
    for _ in range(3):
        c.forward(jx)
        c.backward(jx)
        dev.sync()
        runs.append([x.clone() for x in (c.o, c.lse, c.dq, c.dk, c.dv)])
    for r in runs[1:]:
        assert all(bool((a == b).all()) for a, b in zip(runs[0], r))


def test_slices_of_one_projection(jx, dev):
    """q, k, v and their gradients as slices of one buffer, as a model's projection gives them."""
    t = dev.torch
    c = Case(dev, [300, 21], [300, 21], 4, 2, 64)
    qkv = t.cat([x.flatten(1) for x in (c.q, c.k, c.v)], 1).contiguous()
    grad = t.zeros_like(qkv)
    cut = lambda m: (m[:, :256].unflatten(1, (4, 64)), m[:, 256:384].unflatten(1, (2, 64)),
                     m[:, 384:].unflatten(1, (2, 64)))
    c.q, c.k, c.v = cut(qkv)
    c.dq, c.dk, c.dv = cut(grad)
    c.forward(jx)
    c.check_forward()
    c.backward(jx)
    c.check_backward()


@pytest.mark.parametrize("q_lens,k_lens", [([260, 40], [260, 40]), ([1, 1, 1], [900, 33, 400])])
def test_captured_and_replayed(jx, dev, q_lens, k_lens):
    """Two graphs and an eager call take turns on inputs that change in between."""
    t = dev.torch
    cs = [Case(dev, q_lens, k_lens, 4, 2, 64, seed=s) for s in (1, 2)]
    graphs = []
    for c in cs:
        c.forward(jx)
        c.backward(jx)
        dev.sync()
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g):
            c.forward(jx)
            c.backward(jx)
        graphs.append(g)
    for c in cs:
        for x in (c.q, c.k, c.v, c.dout):
            x.mul_(0.75)
        for x in (c.o, c.dq, c.dk, c.dv):
            x.fill_(7.0)
    for g in graphs + graphs:
        g.replay()
    for c in cs:
        c.check_forward()
        c.check_backward()


def test_two_streams_at_once(jx, dev):
    t = dev.torch
    cs = [Case(dev, [500], [500], 4, 2, 64, seed=s) for s in range(4)]
    dev.sync()
    streams = [t.cuda.Stream() for _ in cs]
    for _ in range(3):
        for c, st in zip(cs, streams):
            c.forward(jx, stream=st.cuda_stream)
            c.backward(jx, stream=st.cuda_stream)
    dev.sync()
    for c in cs:
        c.check_forward()
        c.check_backward()


def test_offsets_outside_are_reported(jx, dev):
    """Offsets behind the tensors' ends or decreasing are taken as the nearest valid ones, and set the error word."""
    jx.device_status()
    for bad in ([0, 300], [0, -5], [90, 40], [-7, 100]):
        c = Case(dev, [100], [100], 2, 1, 64)
        c.cu_q.copy_(c.t.tensor(bad, dtype=c.t.int32))
        c.cu_k.copy_(c.t.tensor(bad, dtype=c.t.int32))
        c.forward(jx)
        assert jx.device_status() == jx.DEVERR_RANGE
        c.backward(jx)
        assert jx.device_status() == jx.DEVERR_RANGE
    c = Case(dev, [100], [100], 2, 1, 64)
    c.forward(jx)
    c.check_forward()
    assert jx.device_status() == 0


def test_a_layer_of_a_transformer(jx, dev):
    """Layer norm, attention on its output, their gradients, clipping and Adam in one run: a training step's part,
    with q = k = v = the normed rows (one head), against the same in 64 bits by automatic differentiation."""
    import ctypes as C
    t = dev.torch
    rows, dim, lens = 330, 64, [100, 230]
    c = Case(dev, lens, lens, 1, 1, dim)
    x = t.randn(rows, dim, generator=c.gen, device="cuda")
    gamma, beta = 1 + 0.1 * t.randn(dim, device="cuda"), 0.1 * t.randn(dim, device="cuda")
    y, mean, rstd = dev.empty((rows, dim)), dev.empty((rows,)), dev.empty((rows,))
    jx.layernorm(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), rows, dim, 1e-5, mean.data_ptr(),
                 rstd.data_ptr(), stream=dev.stream)
    c.q = c.k = c.v = y.view(rows, 1, dim)
    c.forward(jx)
    c.backward(jx)
    dy = dev.empty((rows, dim))
    jx.binary("add", c.dq.data_ptr(), (rows * dim,), c.dk.data_ptr(), (rows * dim,), dy.data_ptr(), dev.stream)
    jx.binary("add", dy.data_ptr(), (rows * dim,), c.dv.data_ptr(), (rows * dim,), dy.data_ptr(), dev.stream)
    dx, dg, db = dev.empty((rows, dim)), dev.empty((dim,)), dev.empty((dim,))
    jx.layernorm_bwd(dy.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
                     dg.data_ptr(), db.data_ptr(), rows, dim, stream=dev.stream)
    # the same in 64 bits
    xs = [v.double().requires_grad_() for v in (x, gamma, beta)]
    n = t.nn.functional.layer_norm(xs[0], (dim,), xs[1], xs[2], 1e-5)
    out = []
    for a, b in ((0, 100), (100, 330)):
        s = (n[a:b] @ n[a:b].t() * c.scale).masked_fill(
            t.ones(b - a, b - a, dtype=t.bool, device="cuda").triu(1), -math.inf)
        out.append(t.softmax(s, 1) @ n[a:b])
    want = t.autograd.grad(t.cat(out), xs, c.dout[:, 0].double())
    for got, w in zip((dx, dg, db), want):
        assert float((got.double() - w).norm()) <= 2e-5 * float(w.norm())
    # clipped to half its norm, then one Adam step: weights move by at most lr
    norm = math.sqrt(float(dg.double().square().sum() + db.double().square().sum()))
    tab = (C.c_void_p * 2)(dg.data_ptr(), db.data_ptr())
    n2 = (C.c_int64 * 2)(dim, dim)
    jx.clip_grads(tab, tab, n2, 2, norm / 2, None, stream=dev.stream)
    assert abs(math.sqrt(float(dg.double().square().sum() + db.double().square().sum())) - norm / 2) <= 1e-5 * norm
    ps = [gamma.clone(), beta.clone()]
    zeros = [dev.full((dim,), 0.0) for _ in range(4)]
    arr = lambda ts: (C.c_void_p * 2)(*[v.data_ptr() for v in ts])
    jx.call("jx_adam_step_f32", arr(ps), tab, arr(zeros[:2]), arr(zeros[2:]), n2, 2, 1e-3, 0.9, 0.999, 1e-8, 1,
            dev.stream)
    for p, before in zip(ps, (gamma, beta)):
        assert 0 < float((p - before).abs().max()) <= 1.01e-3
