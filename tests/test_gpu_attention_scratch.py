"""Attention's scratch over thousands of short sequences, whose 128-row tiles would be nearly empty: the device's pool
is watched for the most that it held.  Outputs against the same call by rings and rows (plain f32, which the tests of
test_gpu_attention.py hold to 64 bits) with the norms' bound of that file, 1e-5, for each side."""
import ctypes as C

import pytest

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu

USED_HIGH = 8  # CU_MEMPOOL_ATTR_USED_MEM_HIGH
LIMIT = (2 << 30) + (256 << 20)  # what a call may take, and some room for statistics and joined parts


class Pool:
    """The most bytes in use of the device's default memory pool, where the library's scratch comes from."""

    def __init__(self, dev):
        dev.torch.cuda.current_stream().synchronize()
        self.cu = C.CDLL("libcuda.so.1")
        self.pool = C.c_void_p()
        assert self.cu.cuDeviceGetDefaultMemPool(C.byref(self.pool), dev.torch.cuda.current_device()) == 0
        assert self.cu.cuMemPoolSetAttribute(self.pool, USED_HIGH, C.byref(C.c_uint64(0))) == 0

    def high(self):
        v = C.c_uint64(0)
        assert self.cu.cuMemPoolGetAttribute(self.pool, USED_HIGH, C.byref(v)) == 0
        return v.value


def outputs(c, jx, **hints):
    for x in (c.o, c.lse, c.dq, c.dk, c.dv):
        x.fill_(7.0)
    c.forward(jx, **hints)
    c.backward(jx, **hints)
    return [x.clone() for x in (c.o, c.lse, c.dq, c.dk, c.dv)]


@pytest.mark.parametrize("count,heads,kv_heads,dim", [
    (2200, 32, 8, 128),  # key heads in groups
    (5000, 24, 8, 64),
    (14000, 2, 1, 128),  # one key head's tiles are beyond the limit already
    (9000, 8, 1, 128),
])
def test_many_short_sequences_and_a_long_one(jx, dev, count, heads, kv_heads, dim):
    t = dev.torch
    lens = [1 + (7 * i * i + 3 * i) % 16 for i in range(count)] + [300]
    c = Case(dev, lens, lens, heads, kv_heads, dim, pad=4, tail=3)
    want = outputs(c, jx, max_q=1, max_k=1)
    dev.sync()
    pool = Pool(dev)
    before = pool.high()
    got = outputs(c, jx)
    dev.sync()
    assert pool.high() - before <= LIMIT
    for x, y in zip(got, want):
        assert float((x.double() - y.double()).norm()) <= 2e-5 * float(y.double().norm())
    assert bool((c.o[-3:] == 7).all()) and bool((c.dq[-3:] == 7).all()) and bool((c.dk[-3:] == 7).all())
    assert jx.device_status() == 0
