"""Refusals of the transformer operators, before any device work (no GPU needed)."""
import ctypes as C

import pytest


def _refused(jx, match, name, *args):
    with pytest.raises(jx.JaxRsError, match=match) as e:
        jx.call(name, *args)
    assert e.value.status == jx.JX_EINVAL


def test_layernorm_refusals(jx):
    f = "jx_layernorm_f32"
    _refused(jx, "bad size", f, 1, 1, 1, 2, None, None, -1, 4, 4, 4, 1e-5, None)
    _refused(jx, "bad size", f, 1, 1, 1, 2, None, None, 1, 0, 4, 4, 1e-5, None)
    _refused(jx, "row stride", f, 1, 1, 1, 2, None, None, 1, 4, 3, 4, 1e-5, None)
    _refused(jx, "row stride", f, 1, 1, 1, 2, None, None, 1, 4, 4, 3, 1e-5, None)
    _refused(jx, "epsilon", f, 1, 1, 1, 2, None, None, 1, 4, 4, 4, -1.0, None)
    _refused(jx, "epsilon", f, 1, 1, 1, 2, None, None, 1, 4, 4, 4, float("nan"), None)
    _refused(jx, "NULL", f, None, 1, 1, 2, None, None, 1, 4, 4, 4, 1e-5, None)
    _refused(jx, "NULL", f, 1, 1, 1, None, None, None, 1, 4, 4, 4, 1e-5, None)
    _refused(jx, "in place", f, 1, 1, 1, 1, None, None, 1, 4, 4, 5, 1e-5, None)
    jx.layernorm(None, None, None, None, 0, 4)  # no rows


def test_layernorm_bwd_refusals(jx):
    f = "jx_layernorm_bwd_f32"
    _refused(jx, "bad size", f, 1, 2, 3, 4, 5, 6, 7, 8, -1, 4, 4, 4, 4, None)
    _refused(jx, "row stride", f, 1, 2, 3, 4, 5, 6, 7, 8, 1, 4, 3, 4, 4, None)
    _refused(jx, "row stride", f, 1, 2, 3, 4, 5, 6, 7, 8, 1, 4, 4, 3, 4, None)
    _refused(jx, "row stride", f, 1, 2, 3, 4, 5, 6, 7, 8, 1, 4, 4, 4, 3, None)
    _refused(jx, "NULL", f, 1, 2, 3, None, 5, 6, 7, 8, 1, 4, 4, 4, 4, None)
    _refused(jx, "dx must not be x", f, 1, 2, 3, 4, 5, 2, 7, 8, 1, 4, 4, 4, 4, None)
    _refused(jx, "in place", f, 1, 2, 3, 4, 5, 1, 7, 8, 1, 4, 4, 4, 5, None)


_GOOD = dict(batch=1, total_q=4, total_k=4, max_q=4, max_k=4, heads=4, kv_heads=2, head_dim=8, ldq=32, ldk=16, ldv=16,
             ldo=32, scale=1.0, causal=1)


@pytest.mark.parametrize("bad,match", [
    (dict(batch=-1), "batch"), (dict(total_q=-1), "total_q"), (dict(total_k=1 << 31), "total_k"),
    (dict(max_q=-1), "max_q"), (dict(max_k=-2), "max_k"), (dict(heads=3), "multiple of kv_heads"),
    (dict(kv_heads=0), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=129, ldq=1000, ldk=1000, ldv=1000, ldo=1000), "head_dim"),
    (dict(ldq=31), "row stride"), (dict(ldk=15), "row stride"), (dict(ldv=15), "row stride"),
    (dict(ldo=31), "row stride"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
])
def test_attention_refusals(jx, bad, match):
    a = {**_GOOD, **bad}
    for name, pointers in (("jx_attention_f32", 7), ("jx_attention_bwd_f32", 11)):
        _refused(jx, match, name, *([16] * pointers), *a.values(), None)


def test_attention_null_pointers_and_empty_calls(jx):
    for name, pointers, may in (("jx_attention_f32", 7, (4,)), ("jx_attention_bwd_f32", 11, ())):
        for i in range(pointers):
            if i not in may:
                p = [16] * pointers
                p[i] = None
                _refused(jx, "NULL", name, *p, *_GOOD.values(), None)
        none = {**_GOOD, "total_q": 0, "total_k": 0}
        jx.call(name, *([None] * pointers), *none.values(), None)
        jx.call(name, *([None] * pointers), *{**_GOOD, "batch": 0}.values(), None)


def test_clip_refusals(jx):
    p = (C.c_void_p * 2)(16, 16)
    n = (C.c_int64 * 2)(3, 5)
    with pytest.raises(jx.JaxRsError, match="negative tensor count"):
        jx.clip_grads(p, p, n, -1, 1.0)
    with pytest.raises(jx.JaxRsError, match="negative size"):
        jx.clip_grads(p, p, (C.c_int64 * 2)(3, -5), 2, 1.0)
    with pytest.raises(jx.JaxRsError, match="tensor 1 has a NULL pointer"):
        jx.clip_grads((C.c_void_p * 2)(16, None), p, n, 2, 1.0)
    with pytest.raises(jx.JaxRsError, match="tensor 0 has a NULL pointer"):
        jx.clip_grads(p, (C.c_void_p * 2)(None, 16), n, 2, 1.0)
    with pytest.raises(jx.JaxRsError, match="NULL array"):
        jx.clip_grads(p, None, n, 2, 1.0)
    with pytest.raises(jx.JaxRsError, match="max_norm"):
        jx.clip_grads(p, p, n, 2, -1.0)
    with pytest.raises(jx.JaxRsError, match="max_norm"):
        jx.clip_grads(p, p, n, 2, float("nan"))
    with pytest.raises(jx.JaxRsError, match="NULL pointer"):
        jx.grad_norm(p, n, 2, None)
    with pytest.raises(jx.JaxRsError, match="too many tensors"):
        jx.grad_norm(p, n, (1 << 20) + 1, 16)


def test_attention_outputs_apart_from_inputs(jx):
    size = [*_GOOD.values(), None]
    good = [16 * (i + 1) for i in range(7)]  # q, k, v, o, lse, cu_q, cu_k
    for i in (0, 1, 2):
        p = list(good)
        p[3] = p[i]
        _refused(jx, "must not be an input", "jx_attention_f32", *p, *size)
    good = [16 * (i + 1) for i in range(11)]  # q, k, v, o, lse, dout, dq, dk, dv, cu_q, cu_k
    for i in range(6):
        for j in (6, 7, 8):
            p = list(good)
            p[j] = p[i]
            _refused(jx, "must not be an input", "jx_attention_bwd_f32", *p, *size)
    for i, j in ((6, 7), (7, 8), (6, 8)):
        p = list(good)
        p[j] = p[i]
        _refused(jx, "different tensors", "jx_attention_bwd_f32", *p, *size)
