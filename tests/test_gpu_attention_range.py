"""Attention where an operand's rows or columns differ widely in size: each column, and each row, against its own
magnitude.  Tolerances as in test_gpu_attention.py: the forward pass element by element, the gradients' norms by column
or by row (64 values at least, as independent as those of a whole tensor) with ||error|| <= 2e-6 ||mag|| + 1e-5 ||want||."""
import pytest

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


def check(c, dims, rows=slice(None), keys=slice(None)):
    """Norms over `dims` of the gradients of [tokens, heads, dim]."""
    _, _, _, g, m = c.reference(True)
    for name, got, want, mag in zip(("dq", "dk", "dv"), (c.dq, c.dk, c.dv), g, m):
        at = rows if name == "dq" else keys
        n = lambda x: x[at].double().norm(dim=dims)
        share = n(got.double() - want) / (2e-6 * n(mag) + 1e-5 * n(want) + 1e-300)
        assert float(share.max()) <= 1, (name, float(share.max()), int(share.argmax()))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", [12, 20, 25])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_one_large_column(jx, dev, dim, power, which):
    """A column 2^power times the others, which no row's largest value shows; scores stay as they were."""
    c = Case(dev, [300], [300], 2, 1, dim)
    getattr(c, which)[:, :, 0] *= 2.0 ** power
    if which in ("q", "k"):
        (c.k if which == "q" else c.q)[:, :, 0] *= 2.0 ** -power
    c.forward(jx)
    c.check_forward()
    c.backward(jx)
    check(c, 0)
    assert jx.device_status() == 0


ROWS = [(64, 256, True), (64, 2048, True), (64, 2048, False), (64, 8192, True), (128, 256, True), (128, 700, False),
        (128, 2048, True), (128, 8192, True)]


@pytest.mark.parametrize("dim,n,causal", ROWS)
@pytest.mark.parametrize("power", [4, 7, 10, 14, 19])
def test_few_large_rows_of_dout(jx, dev, dim, n, causal, power):
    """One token in 128 with a gradient 2^power times the others': dq of the others, dk and dv of the keys that only
    others see (the last ones of a causal sequence)."""
    c = Case(dev, [n], [n], 2, 1, dim, causal)
    c.dout[3::128] *= 2.0 ** power
    c.forward(jx)
    c.backward(jx)
    check(c, (1, 2))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_lens,k_lens", [([1000], [1000]), ([130, 300, 77], [130, 500, 200]), ([400], [250])])
def test_rows_of_dout_of_all_sizes(jx, dev, dim, q_lens, k_lens):
    """Tokens that are predicted well and badly, in any order, heads sharing keys."""
    c = Case(dev, q_lens, k_lens, 6, 2, dim)
    t = dev.torch
    c.dout *= 2.0 ** -t.randint(0, 20, (c.tq, 1, 1), device="cuda", generator=c.gen).float()
    c.forward(jx)
    c.backward(jx)
    check(c, (1, 2))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("zero", [slice(0, 128), slice(0, 200), slice(130, 200)])
def test_tiles_of_zero_gradient_and_large_values(jx, dev, dim, zero):
    """dout of zero gives gradients of zero, however large v is."""
    c = Case(dev, [200], [200], 2, 1, dim)
    c.v *= 1e32
    c.dout *= 1e-3
    c.dout[zero] = 0.0
    c.forward(jx)
    c.backward(jx)
    assert bool((c.dq[zero] == 0).all())
    check(c, (1, 2))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_all_sizes(jx, dev, dim, which, causal):
    """Rows of one operand over 2^19, large ones behind small ones and before them."""
    c = Case(dev, [130, 700], [400, 700], 4, 2, dim, causal)
    t, x = dev.torch, getattr(c, which)
    x *= 2.0 ** -t.randint(0, 20, (x.shape[0], 1, 1), device="cuda", generator=c.gen).float()
    x[3::128] *= 2.0 ** 4
    c.forward(jx)
    c.check_forward()
    c.backward(jx)
    check(c, (1, 2))
