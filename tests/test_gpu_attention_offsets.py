"""Packed offsets outside their tensors: each is taken as the nearest one inside and reported, by every kernel alike."""
import pytest

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu

# hints under which the forward pass and the gradients go by tiles, and by rings and rows
HINTS = [(100000, 100000), (1, 1)]


def moved(c, cu, first, last):
    """`cu` with its first offsets and its last one moved outside."""
    at = cu.tolist()
    at[:len(first)] = first
    at[-1] += last
    return c.t.tensor(at, dtype=c.t.int32, device="cuda")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("q_lens,k_lens,first_q,first_k,last", [
    ([100], [300], [-7], [-7], 0), ([100], [300], [0], [-(1 << 31)], 0), ([100], [300], [-1], [0], 1000),
    ([0, 260, 40], [0, 130, 370], [-300, -7], [-5, -2], 5), ([0, 0, 200], [0, 0, 140], [-400, -200, -1], [0, 0, 0], 0),
])
def test_offsets_outside_are_taken_inside(jx, dev, q_lens, k_lens, first_q, first_k, last, hint, causal):
    c = Case(dev, q_lens, k_lens, 4, 2, 64, causal)
    c.cu_q, c.cu_k = moved(c, c.cu_q, first_q, last), moved(c, c.cu_k, first_k, last)
    jx.device_status()
    c.forward(jx, max_q=hint[0], max_k=hint[1])
    c.check_forward()
    assert jx.device_status() == jx.DEVERR_RANGE
    c.backward(jx, max_q=hint[0], max_k=hint[1])
    c.check_backward()
    assert jx.device_status() == jx.DEVERR_RANGE


def test_gradients_in_parts_with_an_offset_outside(jx, dev):
    """One key head: a tile's query rows are cut into parts, and a launch of its own joins them."""
    c = Case(dev, [1500], [1500], 4, 1, 64)
    c.cu_k = moved(c, c.cu_k, [-200], 0)
    c.forward(jx)
    c.check_forward()
    c.backward(jx)
    c.check_backward()
    assert jx.device_status() == jx.DEVERR_RANGE
