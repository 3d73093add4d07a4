"""Layer norm's gradient for rows whose mean times 1 / sqrt(var + eps) is beyond f32 although no column's xhat is."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [3, 100, 101, 250, 300, 500, 600, 700, 1000, 1111, 1500, 2000, 3000, 3001, 6000, 6001,
                                  12000, 12001, 17000])
def test_a_constant_row_of_large_values(jx, dev, cols):
    """xhat is zero, and dx = (dy - mean(dy)) rstd.  Two subtractions, a product and a sum of cols terms whose
    rounding is at most (cols / 32 + 32) 2^-24 of the largest |dy|, however the threads share it."""
    t = dev.torch
    rows, value, rstd_value = 5, 1.2e36, 1e-5 ** -0.5
    gen = t.Generator(device="cuda").manual_seed(cols)
    x = t.full((rows, cols), value, device="cuda")
    dy = t.randn((rows, cols), generator=gen, device="cuda")
    mean, rstd = t.full((rows,), value, device="cuda"), t.full((rows,), rstd_value, device="cuda")
    assert value * rstd_value > t.finfo(t.float32).max
    dx, dg, db = dev.empty((rows, cols)), dev.empty((cols,)), dev.empty((cols,))
    jx.layernorm_bwd(dy.data_ptr(), x.data_ptr(), None, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
                     dg.data_ptr(), db.data_ptr(), rows, cols, stream=dev.stream)
    d = dy.double()
    want = (d - d.mean(1, keepdim=True)) * float(rstd[0])
    u = 2.0 ** -24
    assert float((dx.double() - want).abs().max()) <= (cols / 32 + 64) * u * float(d.abs().max()) * float(rstd[0])
    assert bool((dg == 0).all())
    assert float((db.double() - d.sum(0)).abs().max()) <= rows * u * float(d.abs().sum(0).max())
