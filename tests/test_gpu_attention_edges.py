"""Attention at the edges of its kernels: every kernel at every length, values that the scaled operands do not
serve, unusual scales, offsets beyond 32 bits, and how far non-finite values reach.  Tolerances as in
test_gpu_attention.py."""
import math

import pytest

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu

SHORT = [([1], [1], 1, 1, 64), ([1], [1], 3, 1, 128), ([2, 0, 5], [2, 3, 1], 4, 2, 100), ([17], [17], 2, 2, 33),
         ([1, 1, 1], [129, 0, 64], 8, 1, 128), ([31, 33], [63, 65], 2, 1, 64)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim", SHORT)
@pytest.mark.parametrize("hint", [(100000, 100000), (0, 0), (3, 100), (1, 1 << 40)])
def test_short_lengths_on_every_kernel(jx, dev, q_lens, k_lens, heads, kv_heads, dim, causal, hint):
    """The hints choose the kernel: tiles, rings of each width, rows."""
    c = Case(dev, q_lens, k_lens, heads, kv_heads, dim, causal, pad=2, tail=1)
    c.forward(jx, max_q=hint[0], max_k=hint[1])
    c.check_forward()
    c.backward(jx, max_q=hint[0], max_k=hint[1])
    c.check_backward()
    assert jx.device_status() == 0


@pytest.mark.parametrize("heads,kv_heads,lens", [(64, 1, [1, 1]), (40, 2, [2, 1]), (24, 1, [5]), (33, 1, [1]),
                                                 (16, 8, [30]), (128, 1, [1])])
@pytest.mark.parametrize("dim", [64, 128, 90])
def test_many_rows_per_key_head(jx, dev, heads, kv_heads, lens, dim):
    """More rows per key head than one pass of the rings takes."""
    c = Case(dev, lens, [n + 700 for n in lens], heads, kv_heads, dim)
    c.forward(jx)
    c.check_forward()


@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim", [
    ([1], [16384], 1, 1, 128), ([1], [4100], 1, 1, 33), ([2, 4, 4, 1], [10194, 17, 30, 4], 2, 1, 127),
    ([4], [14400], 4, 4, 128), ([1, 3], [5, 6000], 3, 1, 64)])
def test_many_pieces_of_a_head(jx, dev, q_lens, k_lens, heads, kv_heads, dim):
    """Long histories of few heads: hundreds of rings share a head, and one block joins their pieces."""
    c = Case(dev, q_lens, k_lens, heads, kv_heads, dim)
    c.forward(jx)
    c.check_forward()


@pytest.mark.parametrize("q_lens,k_lens", [([40000], [0]), ([5], [7]), ([300, 2], [0, 400])])
def test_hints_beyond_the_tensors(jx, dev, q_lens, k_lens):
    """A hint costs no launches for rows that are not there, and rows without keys none of their own."""
    c = Case(dev, q_lens, k_lens, 8, 2, 64)
    c.forward(jx, max_q=1 << 62, max_k=1 << 62)
    c.check_forward()
    c.backward(jx, max_q=1 << 62, max_k=1 << 62)
    c.check_backward()
    assert jx.device_status() == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,n", [(1, 1, 3000), (4, 1, 1500), (6, 3, 700)])
def test_gradient_in_parts(jx, dev, dim, causal, heads, kv_heads, n):
    """Few key tiles: each one's query rows are cut into parts."""
    c = Case(dev, [n, 65], [n, 190], heads, kv_heads, dim, causal, pad=1)
    c.forward(jx)
    c.backward(jx)
    c.check_backward()


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0, 3.0])
@pytest.mark.parametrize("q_lens,k_lens", [([150], [150]), ([1, 2], [300, 40])])
def test_scales(jx, dev, scale, q_lens, k_lens):
    c = Case(dev, q_lens, k_lens, 4, 2, 64, spread=0.5)
    c.scale = scale
    c.forward(jx)
    o, lse, _ = c.reference()
    # the bound of test_gpu_attention takes the scores' magnitude with its sign: norms here
    assert float((c.o.double() - o).norm()) <= 1e-5 * float(o.norm())
    assert float((c.lse.double() - lse).abs().max()) <= 1e-5 * (1 + float(lse.abs().max()))
    c.backward(jx)
    _, _, _, g, m = c.reference(True)
    for got, want, mag in zip((c.dq, c.dk, c.dv), g, m):
        assert float((got.double() - want).norm()) <= 2e-6 * float(mag.abs().norm()) + 1e-5 * float(want.norm())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_rows_of_very_different_sizes(jx, dev, dim, which):
    """A row 2^24 times the others (beyond the tiles' common scale): the gradients of the others keep their precision,
    judged row by row against their own magnitudes."""
    c = Case(dev, [300], [300], 2, 1, dim, spread=0.05)
    x = getattr(c, which)
    if which in ("q", "k"):
        x[200] = 0.0
        x[200, :, 0] = 2.0 ** 24
        (c.k if which == "q" else c.q)[:, :, 0] *= 2.0 ** -24
    else:
        x[200] *= 2.0 ** 24
    c.forward(jx)
    c.backward(jx)
    _, _, _, g, m = c.reference(True)
    for got, want, mag in zip((c.dq, c.dk, c.dv), g, m):
        off = (got.double() - want).flatten(1).norm(dim=1)
        assert bool((off <= 5e-6 * mag.flatten(1).norm(dim=1) + 2e-5 * want.flatten(1).norm(dim=1) + 1e-30).all())


@pytest.mark.parametrize("size", [1e-30, 1e-10, 1e10])
def test_gradients_of_any_size(jx, dev, size):
    """dout scales every gradient; zero rows (tokens that the loss leaves out) among them."""
    c = Case(dev, [140, 20], [140, 300], 2, 1, 128)
    c.dout.mul_(size)
    c.dout[10:30] = 0.0
    c.forward(jx)
    c.backward(jx)
    c.check_backward()


@pytest.mark.parametrize("dim", [64, 128])
def test_non_finite_values_stay_with_the_rows_that_see_them(jx, dev, dim):
    t = dev.torch
    c = Case(dev, [200, 150], [200, 150], 2, 1, dim, tail=4, head=2)
    for x in (c.q, c.k, c.v, c.dout):
        x[:2], x[-4:] = float("nan"), float("inf")
    c.forward(jx)
    c.backward(jx)
    c.check_forward()
    c.check_backward()
    clean = [x.clone() for x in (c.o, c.dq, c.dk, c.dv)]
    a, b = c.cq[1], c.cq[2]  # the second sequence
    c.v[a - 1] = float("nan")  # the first sequence's last key, seen by its last row alone
    c.forward(jx)
    c.backward(jx)
    assert bool(t.isnan(c.o[a - 1]).all()) and bool(t.isnan(c.dq[a - 1]).all())
    for got, want in ((c.o, clean[0]), (c.dq, clean[1])):
        assert float((got[2:a - 1] - want[2:a - 1]).abs().max()) <= 1e-5 * float(want[2:a - 1].abs().max())
    for got, want in zip((c.o, c.dq, c.dk, c.dv), clean):
        assert bool((got[a:b] == want[a:b]).all())  # the other sequence: the same bits


def test_one_row_of_dout_non_finite(jx, dev):
    """Its own dq, and the keys that it sees."""
    t = dev.torch
    c = Case(dev, [260], [260], 1, 1, 64)
    c.forward(jx)
    c.backward(jx)
    clean = [x.clone() for x in (c.dq, c.dk, c.dv)]
    c.dout[130] = float("inf")
    c.backward(jx)
    keep = [r for r in range(260) if r != 130]
    assert float((c.dq[keep] - clean[0][keep]).abs().max()) <= 1e-5 * float(clean[0].abs().max())
    for got, want in zip((c.dk, c.dv), clean[1:]):
        assert bool(t.isfinite(got[131:]).all())
        assert float((got[131:] - want[131:]).abs().max()) <= 1e-5 * float(want.abs().max())
        assert not bool(t.isfinite(got[:131]).any(2).any())


@pytest.mark.parametrize("q_lens,k_lens", [([1], [1090]), ([70], [1090])])
def test_offsets_beyond_32_bits(jx, dev, q_lens, k_lens):
    """Key rows 2^21 elements apart: the last ones lie behind 2^31 elements."""
    t = dev.torch
    c = Case(dev, q_lens, k_lens, 4, 2, 64)
    ld = 1 << 21
    try:
        buf = t.empty(1090 * ld, device="cuda")
    except t.OutOfMemoryError:
        pytest.skip("needs 9 GB")
    at = lambda off: buf.view(1090, ld)[:, off:off + 128].unflatten(1, (2, 64))
    k, v, dk, dv = (at(o) for o in (0, 4096, 8192, 12288))
    k.copy_(c.k)
    v.copy_(c.v)
    c.k, c.v, c.dk, c.dv = k, v, dk, dv
    c.forward(jx)
    c.check_forward()
    c.backward(jx)
    c.check_backward()


def test_many_sequences(jx, dev):
    """More sequences than a warp looks through at a time, empty ones among them."""
    lens = [(7 * i * i + 3 * i) % 61 for i in range(1500)]
    c = Case(dev, lens, lens, 2, 1, 32)
    c.forward(jx)
    c.check_forward()
    c.backward(jx)
    c.check_backward()


@pytest.mark.parametrize("q_lens,k_lens,heads,kv_heads,dim,causal", [
    ([4096], [64], 8, 8, 64, False),     # dq has far more to do than dk and dv
    ([64], [4096], 8, 2, 128, False),    # and far less
    ([3000, 0, 500], [0, 700, 1], 4, 1, 64, False),
    ([2048], [0], 8, 8, 128, True),
    ([1500, 700], [1500, 700], 8, 2, 128, True),
])
def test_what_follows_in_the_stream_sees_everything(jx, dev, q_lens, k_lens, heads, kv_heads, dim, causal):
    """Launches overlap; copies behind a call, without a wait on the host, must still find it complete."""
    t = dev.torch
    c = Case(dev, q_lens, k_lens, heads, kv_heads, dim, causal)
    c.forward(jx)
    outs = (c.o, c.lse, c.dq, c.dk, c.dv)
    c.backward(jx)
    t.cuda.synchronize()
    want = [x.clone() for x in outs]
    for _ in range(5):
        for x in outs:
            x.fill_(math.nan)
        c.forward(jx)
        after = [x.clone() for x in (c.o, c.lse)]
        c.backward(jx)
        after += [x.clone() for x in (c.dq, c.dk, c.dv)]
        t.cuda.synchronize()
        for x, y in zip(after, want):
            assert t.equal(x, y)
    assert jx.device_status() == 0
