"""Cases of the transformer operators: layer norm, packed attention and gradient clipping.

Every operator is here in its plain form, as elementary torch operations in 32 bits (sums over many values in
64), and as the calls that a program makes of the library's entry points (`own`).  `exact` computes the same
outputs from the operators' definitions in 64 bits.

    layer norm   y = (x - mean) / sqrt(var + eps) * gamma + beta over the last axis, biased variance;
                 backward: dx, dgamma, dbeta from dy, x and the rows' mean and 1 / sqrt(var + eps)
    attention    sequences packed one behind the other, query heads sharing key heads in groups; causal masks are
                 aligned at the end of the keys, so that one query behind a long history is a decoding step;
                 o = softmax(scale q k^T) v and the rows' log-sum-exp; backward: dq, dk, dv
    clipping     norm = sqrt(sum of all squares) over many tensors, each scaled by min(1, max_norm / (norm + 1e-6))
"""
import ctypes
import importlib
import math

import torch

own = False

EPS = 1e-5
CLIP_EPS = 1e-6


def listed():
    return [
        # one token's hidden state on its way through a decoder
        {"name": "layernorm one token", "op": "ln_fwd", "rows": 1, "cols": 4096, "pad": 0},
        # a training batch of 16384 tokens
        {"name": "layernorm batch", "op": "ln_fwd", "rows": 16384, "cols": 4096, "pad": 0},
        # a small model's batch with an odd width, rows cut out of a wider buffer
        {"name": "layernorm backward odd", "op": "ln_bwd", "rows": 1000, "cols": 1111, "pad": 5},
        # the gradient of a training batch, with the sums over all rows for the weight and the bias
        {"name": "layernorm backward batch", "op": "ln_bwd", "rows": 16384, "cols": 2048, "pad": 0},
        # one decoding step of eight requests over histories of different lengths
        {"name": "attention one token", "op": "attn_fwd", "q_lens": "1,1,1,1,1,1,1,1",
         "k_lens": "4096,1027,2500,17,3999,640,2048,1", "heads": 32, "kv_heads": 8, "dim": 128, "causal": True,
         "fused": False},
        # four short prompts, q, k and v slices of one projection's output
        {"name": "attention short prompts", "op": "attn_fwd", "q_lens": "100,37,128,1", "k_lens": "100,37,128,1",
         "heads": 8, "kv_heads": 2, "dim": 64, "causal": True, "fused": True},
        # one long prompt
        {"name": "attention long prompt", "op": "attn_fwd", "q_lens": "8192", "k_lens": "8192", "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": True, "fused": False},
        # prompts of different lengths behind cached histories, packed
        {"name": "attention packed prompts", "op": "attn_fwd", "q_lens": "2049,511,1300,64,777,1900",
         "k_lens": "2049,1511,1300,1088,777,2400", "heads": 16, "kv_heads": 4, "dim": 128, "causal": True,
         "fused": False},
        # a packed training batch of documents, the gradients in the layout of the projection's output
        {"name": "attention backward packed", "op": "attn_bwd", "q_lens": "1023,333,2048,130,562",
         "k_lens": "1023,333,2048,130,562", "heads": 16, "kv_heads": 16, "dim": 64, "causal": True, "fused": True},
        # one training sequence with shared key heads
        {"name": "attention backward long", "op": "attn_bwd", "q_lens": "4096", "k_lens": "4096", "heads": 16,
         "kv_heads": 4, "dim": 128, "causal": True, "fused": False},
        # the 48 weights, biases and norms of a small model, a fraction of a megabyte in all
        {"name": "clip small tensors", "op": "clip", "count": 48, "largest": 16384, "smallest": 1, "active": True},
        # five layers' weights and biases of 8192 units
        {"name": "clip large tensors", "op": "clip", "count": 10, "largest": 67108864, "smallest": 8192,
         "active": True},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "attn_fwd", "attn_fwd", "attn_step", "attn_bwd", "attn_bwd", "clip"])
    if op in ("ln_fwd", "ln_bwd"):
        cols = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, min(65536, (1 << 26) // cols))
        return {"op": op, "rows": rows, "cols": cols, "pad": rng.choice([0, 0, 4, 7])}
    if op == "clip":
        return {"op": op, "count": _spread(rng, 1, 400), "largest": _spread(rng, 64, 1 << 20),
                "smallest": rng.choice([0, 1, 17, 64]), "active": rng.random() < 0.75}
    kv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 4, 5, 8])
    dim = rng.choice([16, 32, 40, 64, 64, 72, 80, 96, 127, 128, 128, 128])
    batch = _spread(rng, 1, 16)
    if op == "attn_step":
        k = [_spread(rng, 1, 16384) for _ in range(batch)]
        q = [rng.choice([1, 1, 1, 2, 4]) for _ in range(batch)]
        q = [min(a, b) for a, b in zip(q, k)]
        op = "attn_fwd"
        causal = True
    else:
        longest = _spread(rng, 16, 4096)
        causal = rng.random() < 0.8
        # prompts, behind a history, or with fewer keys than queries: the first rows then see none
        q = [_spread(rng, 1, longest) for _ in range(batch)]
        k = [max(1, a + rng.choice([0, 0, 0, rng.randint(1, 300), -rng.randint(1, 40)])) for a in q]
        while batch * kv * group * max(q) * max(k) > (1 << 30 if op == "attn_fwd" else 1 << 28):
            q, k = [-(-a // 2) for a in q], [-(-a // 2) for a in k]
    return {"op": op, "q_lens": ",".join(map(str, q)), "k_lens": ",".join(map(str, k)), "heads": kv * group,
            "kv_heads": kv, "dim": dim, "causal": causal, "fused": q == k and rng.random() < 0.5}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _lens(text):
    return [int(v) for v in text.split(",")]


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _clip_sizes(case):
    """Sizes spread evenly over the logarithm between the two ends, the largest ones as often as the smallest."""
    n, lo, hi = case["count"], max(1, case["smallest"]), case["largest"]
    if n == 10 and hi == 8192 * 8192:
        return [hi, lo] * 5
    sizes = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)]
    if case["smallest"] == 0:
        sizes[0] = 0
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)

    s = {"op": case["op"], "case": dict(case)}
    if case["op"] in ("ln_fwd", "ln_bwd"):
        rows, cols, pad = case["rows"], case["cols"], case["pad"]
        # hidden states: columns with offsets and magnitudes of their own
        x = normal(rows, cols + pad) * (0.5 + normal(cols + pad).abs()) + 0.3 * normal(cols + pad)
        s |= {"x": x[:, :cols], "gamma": 1 + 0.1 * normal(cols), "beta": 0.1 * normal(cols)}
        if case["op"] == "ln_fwd":
            s |= {"y": torch.zeros(rows, cols, device="cuda"), "mean": torch.zeros(rows, device="cuda"),
                  "rstd": torch.zeros(rows, device="cuda")}
        else:
            xd = s["x"].double()
            s |= {"dy": (1e-2 * normal(rows, cols + pad))[:, :cols], "mean": xd.mean(1).float(),
                  "rstd": (xd.var(1, unbiased=False) + EPS).rsqrt().float(),
                  "dx": torch.zeros(rows, cols, device="cuda"), "dgamma": torch.zeros(cols, device="cuda"),
                  "dbeta": torch.zeros(cols, device="cuda")}
    elif case["op"] == "clip":
        sizes = _clip_sizes(case)
        offsets = _offsets(sizes)
        flat = normal(offsets[-1]) * 1e-3
        out = torch.zeros_like(flat)
        grads = [flat[a:b] for a, b in zip(offsets, offsets[1:])]
        outs = [out[a:b] for a, b in zip(offsets, offsets[1:])]
        for i, g in enumerate(grads):  # layers whose gradients differ in size
            g.mul_(2.0 ** (i % 7 - 3))
        n = len(sizes)
        norm = float(flat.double().square().sum().sqrt())
        s |= {"grads": grads, "outs": outs, "out": out, "norm": torch.zeros(1, device="cuda"),
              "max_norm": norm * (0.5 if case["active"] else 2.0),
              "grad_table": (ctypes.c_void_p * n)(*[g.data_ptr() for g in grads]),
              "out_table": (ctypes.c_void_p * n)(*[g.data_ptr() for g in outs]),
              "size_table": (ctypes.c_int64 * n)(*sizes)}
    else:
        q_lens, k_lens = _lens(case["q_lens"]), _lens(case["k_lens"])
        H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
        tq, tk = sum(q_lens), sum(k_lens)

        def buffers(make):
            """q, k and v: tensors of their own, or slices of one projection's output."""
            if case["fused"]:
                qkv = make(tq, (H + 2 * Hk) * D)
                return [qkv, qkv[:, :H * D].unflatten(1, (H, D)),
                        qkv[:, H * D:(H + Hk) * D].unflatten(1, (Hk, D)), qkv[:, (H + Hk) * D:].unflatten(1, (Hk, D))]
            return [None, make(tq, H, D), make(tk, Hk, D), make(tk, Hk, D)]

        _, q, k, v = buffers(normal)
        q.mul_(1.5)  # scores with a spread as trained heads have it
        s |= {"q": q, "k": k, "v": v, "scale": 1.0 / math.sqrt(D), "max_q": max(q_lens), "max_k": max(k_lens),
              "cu_q": torch.tensor(_offsets(q_lens), dtype=torch.int32, device="cuda"),
              "cu_k": torch.tensor(_offsets(k_lens), dtype=torch.int32, device="cuda"),
              "o": torch.zeros(tq, H, D, device="cuda"), "lse": torch.zeros(H, tq, device="cuda")}
        if case["op"] == "attn_bwd":
            o, lse = _attention(s)
            s["o"].copy_(o)
            s["lse"].copy_(lse)
            s["do"] = normal(tq, H, D) * 1e-2
            s["dqkv"], s["dq"], s["dk"], s["dv"] = buffers(lambda *shape: torch.zeros(shape, device="cuda"))
    return s


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------
def _layernorm(s):
    x = s["x"]
    mean = x.mean(1)
    c = x - mean[:, None]
    rstd = 1.0 / (c.square().mean(1) + EPS).sqrt()
    return c * rstd[:, None] * s["gamma"] + s["beta"], mean, rstd


def _layernorm_bwd(s):
    xhat = (s["x"] - s["mean"][:, None]) * s["rstd"][:, None]
    g = s["dy"] * s["gamma"]
    dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
    return dx, (s["dy"] * xhat).sum(0), s["dy"].sum(0)


def _padded(s):
    """Rows of each sequence padded to the longest: index tables, their valid places and the scores' mask."""
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    lq, lk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    i = torch.arange(s["max_q"], device="cuda")
    j = torch.arange(s["max_k"], device="cuda")
    in_q, in_k = i < lq[:, None], j < lk[:, None]
    at_q = torch.where(in_q, cu_q[:-1, None] + i, 0)
    at_k = torch.where(in_k, cu_k[:-1, None] + j, 0)
    seen = in_q[:, :, None] & in_k[:, None, :]
    if s["case"]["causal"]:
        seen = seen & (j <= i[:, None] + (lk - lq)[:, None, None])
    return at_q, at_k, in_q, in_k, seen


def _by_head(x, at, kv_heads):
    """[tokens, heads, dim] -> [batch, kv_heads, group * length, dim]."""
    b, n = at.shape
    return x[at].unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, x.shape[2])


def _packed(x, inside, like):
    """[batch, kv_heads, group * length, dim] -> [tokens, heads, dim], `inside` saying which places hold a token."""
    b, n = inside.shape
    hk = x.shape[1]
    x = x.unflatten(2, (-1, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return x[inside].reshape(like.shape)


def _scores(s, q, k, seen):
    group = q.shape[2] // seen.shape[1]
    x = (q @ k.transpose(2, 3)) * s["scale"]
    return x.unflatten(2, (group, -1)).masked_fill_(~seen[:, None, None], -math.inf).flatten(2, 3)


def _attention(s):
    hk = s["k"].shape[1]
    at_q, at_k, in_q, in_k, seen = _padded(s)
    q, k, v = _by_head(s["q"], at_q, hk), _by_head(s["k"], at_k, hk), _by_head(s["v"], at_k, hk)
    x = _scores(s, q, k, seen)
    top = x.amax(3, keepdim=True)
    p = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(3, keepdim=True)
    o = (p @ v) / torch.where(total == 0, 1.0, total)
    lse = _packed(top + total.log(), in_q, s["q"][:, :, :1])
    return _packed(o, in_q, s["q"]), lse[:, :, 0].t().contiguous()


def _attention_bwd(s):
    hk, group = s["k"].shape[1], s["q"].shape[1] // s["k"].shape[1]
    at_q, at_k, in_q, in_k, seen = _padded(s)
    q, k, v = _by_head(s["q"], at_q, hk), _by_head(s["k"], at_k, hk), _by_head(s["v"], at_k, hk)
    o, do = _by_head(s["o"], at_q, hk), _by_head(s["do"], at_q, hk)
    do = do * in_q[:, None, None, :, None].expand(-1, 1, group, -1, 1).flatten(2, 3)
    lse = _by_head(s["lse"].t()[:, :, None], at_q, hk)
    p = (_scores(s, q, k, seen) - torch.where(lse == -math.inf, 0.0, lse)).exp()
    dv = p.transpose(2, 3) @ do
    ds = p * (do @ v.transpose(2, 3) - (do * o).sum(3, keepdim=True)) * s["scale"]
    return (_packed(ds @ k, in_q, s["q"]), _packed(ds.transpose(2, 3) @ q, in_k, s["k"]),
            _packed(dv, in_k, s["v"]))


def _clip(s):
    norm = torch.stack([g.square().sum(dtype=torch.float64) for g in s["grads"]]).sum().sqrt()
    factor = (s["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0).float()
    return torch.cat([g * factor for g in s["grads"]]), norm.float().reshape(1)


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
_package = None


def _jx():
    global _package
    if _package is None:
        _package = importlib.import_module("jax-rs_b200")
        _package.init(0)
    return _package


def _run_own(s):
    jx = _jx()
    st = torch.cuda.current_stream().cuda_stream
    op = s["op"]
    if op == "ln_fwd":
        x, y = s["x"], s["y"]
        jx.layernorm(x.data_ptr(), s["gamma"].data_ptr(), s["beta"].data_ptr(), y.data_ptr(), x.shape[0], x.shape[1],
                     EPS, mean_out=s["mean"].data_ptr(), rstd_out=s["rstd"].data_ptr(), ldx=x.stride(0),
                     ldy=y.stride(0), stream=st)
        return y, s["mean"], s["rstd"]
    if op == "ln_bwd":
        x, dy, dx = s["x"], s["dy"], s["dx"]
        jx.layernorm_bwd(dy.data_ptr(), x.data_ptr(), s["gamma"].data_ptr(), s["mean"].data_ptr(),
                         s["rstd"].data_ptr(), dx.data_ptr(), s["dgamma"].data_ptr(), s["dbeta"].data_ptr(),
                         x.shape[0], x.shape[1], lddy=dy.stride(0), ldx=x.stride(0), lddx=dx.stride(0), stream=st)
        return dx, s["dgamma"], s["dbeta"]
    if op == "clip":
        jx.clip_grads(s["grad_table"], s["out_table"], s["size_table"], len(s["grads"]), s["max_norm"],
                      s["norm"].data_ptr(), stream=st)
        return s["out"], s["norm"]
    q, k, v, o = s["q"], s["k"], s["v"], s["o"]
    shape = dict(batch=s["cu_q"].numel() - 1, total_q=q.shape[0], total_k=k.shape[0], max_q=s["max_q"],
                 max_k=s["max_k"], heads=q.shape[1], kv_heads=k.shape[1], head_dim=q.shape[2], ldq=q.stride(0),
                 ldk=k.stride(0), ldv=v.stride(0), ldo=o.stride(0), scale=s["scale"], causal=s["case"]["causal"],
                 stream=st)
    if op == "attn_fwd":
        jx.attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), s["lse"].data_ptr(),
                     s["cu_q"].data_ptr(), s["cu_k"].data_ptr(), **shape)
        return o, s["lse"]
    jx.attention_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), s["lse"].data_ptr(), s["do"].data_ptr(),
                     s["dq"].data_ptr(), s["dk"].data_ptr(), s["dv"].data_ptr(), s["cu_q"].data_ptr(),
                     s["cu_k"].data_ptr(), **shape)
    return s["dq"], s["dk"], s["dv"]


def run(state):
    if own:
        return _run_own(state)
    return {"ln_fwd": _layernorm, "ln_bwd": _layernorm_bwd, "attn_fwd": _attention, "attn_bwd": _attention_bwd,
            "clip": _clip}[state["op"]](state)


def work(case):
    """Each input read and each output written once; products of visible pairs of rows alone."""
    op = case["op"]
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols = case["rows"], case["cols"]
        if op == "ln_fwd":
            return {"bytes": 4 * (2 * rows * cols + 2 * cols + 2 * rows), "flops": 8 * rows * cols}
        return {"bytes": 4 * (3 * rows * cols + 3 * cols + 2 * rows), "flops": 14 * rows * cols}
    if op == "clip":
        n = sum(_clip_sizes(case))
        return {"bytes": 8 * n + 4, "flops": 3 * n}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    pairs = tq = tk = 0
    for lq, lk in zip(_lens(case["q_lens"]), _lens(case["k_lens"])):
        tq, tk = tq + lq, tk + lk
        if case["causal"]:
            full = max(0, lk - lq)  # keys that every row sees
            n = min(lq, lk)
            pairs += full * lq + n * (n + 1) // 2
        else:
            pairs += lq * lk
    if op == "attn_fwd":
        return {"bytes": 4 * (2 * tq * H * D + 2 * tk * Hk * D + tq * H), "flops": 4 * pairs * H * D}
    return {"bytes": 4 * (4 * tq * H * D + 4 * tk * Hk * D + tq * H), "flops": 10 * pairs * H * D}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "ln_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + EPS) ** -0.5
        y = torch.addcmul(s["beta"].double(), (x - mean.unsqueeze(1)) * rstd.unsqueeze(1), s["gamma"].double())
        return y, mean, rstd
    if op == "ln_bwd":
        x = s["x"].double().requires_grad_()
        gamma = s["gamma"].double().requires_grad_()
        beta = s["beta"].double().requires_grad_()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        y = (x - mean) * (var + EPS) ** -0.5 * gamma + beta
        return torch.autograd.grad(y, (x, gamma, beta), s["dy"].double())
    if op == "clip":
        squares = sum(float((g.double() * g.double()).sum()) for g in s["grads"])
        norm = math.sqrt(squares)
        factor = min(1.0, s["max_norm"] / (norm + CLIP_EPS))
        return torch.cat([g.double() for g in s["grads"]]) * factor, torch.tensor([norm], dtype=torch.float64)
    q_at, k_at = _offsets(_lens(case["q_lens"])), _offsets(_lens(case["k_lens"]))
    H, Hk = case["heads"], case["kv_heads"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((H, s["q"].shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v"))
    for a, b, c, d in zip(q_at, q_at[1:], k_at, k_at[1:]):
        hidden = None
        if case["causal"]:
            hidden = torch.ones(b - a, d - c, dtype=torch.bool, device="cuda").triu_(1 + (d - c) - (b - a))
        for h in range(H):
            g = h // (H // Hk)
            q, k, v = s["q"][a:b, h].double(), s["k"][c:d, g].double(), s["v"][c:d, g].double()
            x = torch.mm(q, k.t()).mul_(s["scale"])
            if hidden is not None:
                x.masked_fill_(hidden, -math.inf)
            total = torch.logsumexp(x, 1)
            p = x.sub_(torch.where(total == -math.inf, 0.0, total)[:, None]).exp_()
            o[a:b, h], lse[h, a:b] = torch.mm(p, v), total
            if op == "attn_bwd":
                do = s["do"][a:b, h].double()
                dv[c:d, g] += torch.mm(p.t(), do)
                dp = torch.mm(do, v.t())
                dx = p * (dp - (dp * p).sum(1, keepdim=True)) * s["scale"]
                dq[a:b, h] = torch.mm(dx, k)
                dk[c:d, g] += torch.mm(dx.t(), q)
    return (o, lse) if op == "attn_fwd" else (dq, dk, dv)
