"""A key cache with room to grow: the room behind a request's keys is a sequence without query rows, whatever it holds."""
import pytest

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,hint", [(1, (1, 1000)), (1, (100000, 100000)), (3, (3, 1000)), (40, (40, 1000)), (1, (0, 0))])
@pytest.mark.parametrize("dim", [64, 128, 90])
def test_room_behind_the_keys(jx, dev, rows, hint, dim):
    t = dev.torch
    capacity, used = 1000, [1, 999, 40, 513, 128, 1000, 700]
    used = [max(n, rows) for n in used]
    q_lens = [n for u in used for n in (rows, 0)]
    k_lens = [n for u in used for n in (u, capacity - u)]
    c = Case(dev, q_lens, k_lens, 8, 2, dim)
    room = t.ones(c.tk, dtype=t.bool, device="cuda")
    for i, u in enumerate(used):
        room[i * capacity:i * capacity + u] = False
    c.k[room], c.v[room] = float("nan"), float("inf")
    c.forward(jx, max_q=hint[0], max_k=hint[1])
    c.check_forward()
    c.backward(jx, max_q=hint[0], max_k=hint[1])
    c.check_backward()
    assert bool((c.dk[room] == 0).all()) and bool((c.dv[room] == 0).all())
    # the next token: one row of room becomes a key
    at = c.cu_k.clone()
    for i, u in enumerate(used):
        if u < capacity:
            at[2 * i + 1] += 1
            c.k[i * capacity + u], c.v[i * capacity + u] = 1.0, -1.0
            c.k_lens[2 * i], c.k_lens[2 * i + 1] = u + 1, capacity - u - 1
    c.cu_k, c.ck = at, at.tolist()
    c.forward(jx, max_q=hint[0], max_k=hint[1])
    c.check_forward()
    assert jx.device_status() == 0
