"""Layer normalisation and cross attention: the cases that are timed, their plain torch forms and
their 64-bit definitions.

The two operators of a decoder layer that reads an encoder's states: the norm in front of it
(forward and backward) and the attention of the decoder's queries over the encoder's keys and
values, whose length is another one than the queries' (forward, its form for single tokens, and
backward).  Tensors lie as the projections before and after them leave them: q and out are
[batch, q_len, q_heads, head_dim], k and v [batch, kv_len, kv_heads, head_dim].

With `own` false `run` computes the plain form, with `own` true it calls the framework.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # The norm in front of one decoding step of eight sequences: latency alone.
        {"name": "norm_step", "op": "norm_fwd", "dtype": "bf16", "params": "f32", "rows": 8, "cols": 1024},
        # The norm over a whole training batch in fp32, the size that the benchmark measures.
        {"name": "norm_fwd_f32", "op": "norm_fwd", "dtype": "f32", "params": "f32", "rows": 65536, "cols": 1024},
        # Its backward pass in mixed precision: bf16 activations, fp32 weights and their gradients.
        {"name": "norm_bwd_bf16", "op": "norm_bwd", "dtype": "bf16", "params": "f32", "rows": 32768, "cols": 1024},
        # Ragged sizes: a packed batch of an odd number of tokens, rows that no vector width divides.
        {"name": "norm_bwd_ragged", "op": "norm_bwd", "dtype": "f32", "params": "f32", "rows": 5003, "cols": 1333},
        # One token of one sequence over its encoder's states: the smallest call, latency counts.
        {"name": "cross_step_one", "op": "cross_step", "dtype": "bf16", "batch": 1, "heads": 16, "kv_heads": 16,
         "q_len": 1, "kv_len": 1500, "dim": 64, "keys": "all"},
        # One token each of a full serving batch with shared key heads over long states.
        {"name": "cross_step_batch", "op": "cross_step", "dtype": "bf16", "batch": 64, "heads": 32, "kv_heads": 8,
         "q_len": 1, "kv_len": 4096, "dim": 128, "keys": "lens"},
        # A training batch: 512 target tokens over 2048 source positions, sources of mixed lengths.
        {"name": "cross_fwd_train", "op": "cross_fwd", "dtype": "bf16", "batch": 16, "heads": 16, "kv_heads": 16,
         "q_len": 512, "kv_len": 2048, "dim": 64, "keys": "lens"},
        # The largest: long targets over longer sources, four query heads to a key head.
        {"name": "cross_fwd_long", "op": "cross_fwd", "dtype": "bf16", "batch": 8, "heads": 16, "kv_heads": 4,
         "q_len": 2048, "kv_len": 4096, "dim": 128, "keys": "all"},
        # fp32, odd lengths, and a mask with holes (dropped source positions).
        {"name": "cross_fwd_f32", "op": "cross_fwd", "dtype": "f32", "batch": 4, "heads": 16, "kv_heads": 16,
         "q_len": 333, "kv_len": 1000, "dim": 64, "keys": "mask"},
        # The backward pass of the training batch.
        {"name": "cross_bwd_train", "op": "cross_bwd", "dtype": "bf16", "batch": 16, "heads": 16, "kv_heads": 16,
         "q_len": 512, "kv_len": 2048, "dim": 64, "keys": "lens"},
        # The backward pass with shared key heads: their gradients are sums over the group.
        {"name": "cross_bwd_shared", "op": "cross_bwd", "dtype": "bf16", "batch": 4, "heads": 16, "kv_heads": 4,
         "q_len": 1024, "kv_len": 2048, "dim": 128, "keys": "lens"},
        # A small fp32 backward pass of odd lengths.
        {"name": "cross_bwd_f32", "op": "cross_bwd", "dtype": "f32", "batch": 2, "heads": 8, "kv_heads": 8,
         "q_len": 77, "kv_len": 300, "dim": 64, "keys": "mask"},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "cross_step", "cross_fwd", "cross_bwd"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op.startswith("norm"):
        cols = rng.choice([_spread(rng, 64, 8192), 8 * _spread(rng, 8, 1024)])
        rows = _spread(rng, 1, min(65536, 67108864 // cols))
        return {"op": op, "dtype": dtype, "params": rng.choice(["f32", dtype]), "rows": rows, "cols": cols}
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    batch = _spread(rng, 1, 64 if op == "cross_step" else 16)
    # (With one key the scores' gradient is zero: a backward pass has some keys to weigh.)
    kv_len = _spread(rng, 16 if op == "cross_bwd" else 1, 8192 if op == "cross_step" else 4096)
    q_len = 1 if op == "cross_step" else _spread(rng, 2, 2048)
    # No drawn case costs more than the largest listed ones.
    most = {"cross_step": 1 << 22, "cross_fwd": 1 << (30 if dtype == "bf16" else 26),
            "cross_bwd": 1 << (27 if dtype == "bf16" else 25)}[op] * 64 // dim
    while batch * heads * q_len * kv_len > most:
        batch, q_len, kv_len = max(1, batch // 2), max(1, q_len * 3 // 4), max(1, kv_len * 3 // 4)
    return {"op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "q_len": q_len,
            "kv_len": kv_len, "dim": dim, "keys": rng.choice(["all", "lens", "mask"])}


def _lens(case):
    """Key counts of the sequences of a batch: from kv_len down to about half of it."""
    b, n = case["batch"], case["kv_len"]
    return [max(1, n - n * i // (2 * b)) for i in range(b)]


def _keys_seen(case):
    """Visible keys over the whole batch."""
    if case["keys"] == "lens":
        return sum(_lens(case))
    n = case["kv_len"]
    return case["batch"] * (n - n // 10 if case["keys"] == "mask" else n)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]

    def normal(*shape, dtype=t):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    if case["op"].startswith("norm"):
        rows, cols, pt = case["rows"], case["cols"], _TYPES[case["params"]]
        # Activations of a residual stream: a scale and an offset of their own in each row.
        x = (normal(rows, cols, dtype=torch.float32) * (0.5 + normal(rows, 1, dtype=torch.float32).abs())
             + normal(rows, 1, dtype=torch.float32)).to(t)
        s = {"case": case, "x": x, "gamma": (1 + 0.1 * normal(cols, dtype=torch.float32)).to(pt)}
        if case["op"] == "norm_fwd":
            s["beta"] = (0.1 * normal(cols, dtype=torch.float32)).to(pt)
        else:
            s["dout"] = normal(rows, cols)
            wide = x.double()  # the row statistics that the forward pass kept
            mean = wide.mean(1)
            s["mean"] = mean.float()
            s["rstd"] = (((wide - mean[:, None]) ** 2).mean(1) + EPS).rsqrt().float()
        return s

    b, n = case["batch"], case["kv_len"]
    s = {"case": case, "lens": None, "mask": None,
         "q": normal(b, case["q_len"], case["heads"], case["dim"]),
         "k": normal(b, n, case["kv_heads"], case["dim"]),
         "v": normal(b, n, case["kv_heads"], case["dim"])}
    if case["keys"] == "lens":
        order = torch.randperm(b, generator=g, device="cuda")
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")[order].contiguous()
    elif case["keys"] == "mask":
        place = torch.rand((b, n), generator=g, device="cuda").argsort(1)
        s["mask"] = (place >= n // 10).to(torch.uint8)
    if case["op"] == "cross_bwd":
        s["dout"] = normal(b, case["q_len"], case["heads"], case["dim"])
        s["out"], s["lse"] = _plain_forward(s)
    return s


# ---- plain forms ----------------------------------------------------------------------------
def _visible(s):
    """[batch, 1, 1, kv_len] truth values."""
    b, n = s["case"]["batch"], s["case"]["kv_len"]
    at = torch.arange(n, device="cuda")
    if s["lens"] is not None:
        return (at[None, :] < s["lens"][:, None])[:, None, None, :]
    if s["mask"] is not None:
        return (s["mask"] != 0)[:, None, None, :]
    return torch.ones((b, 1, 1, n), dtype=torch.bool, device="cuda")


def _by_key_head(x, kv_heads):
    """[batch, len, heads, dim] -> fp32 [batch, kv_heads, group * len, dim]."""
    b, n, h, d = x.shape
    return x.float().permute(0, 2, 1, 3).reshape(b, kv_heads, h // kv_heads * n, d)


def _by_token(x, n, heads):
    """The way back."""
    b, _, _, d = x.shape
    return x.reshape(b, heads, n, d).permute(0, 2, 1, 3).contiguous()


def _plain_scores(s):
    case = s["case"]
    q, k = _by_key_head(s["q"], case["kv_heads"]), _by_key_head(s["k"], case["kv_heads"])
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(case["dim"])
    return torch.where(_visible(s), scores, -math.inf)


def _plain_forward(s):
    case = s["case"]
    scores = _plain_scores(s)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _by_key_head(s["v"], case["kv_heads"])) / total
    lse = (top + torch.log(total)).reshape(case["batch"], case["heads"], case["q_len"])
    return _by_token(out, case["q_len"], case["heads"]).to(s["q"].dtype), lse


def _plain_backward(s):
    case = s["case"]
    hk = case["kv_heads"]
    q, k, v = (_by_key_head(s[n], hk) for n in ("q", "k", "v"))
    do, o = _by_key_head(s["dout"], hk), _by_key_head(s["out"], hk)
    p = torch.exp(_plain_scores(s) - s["lse"].reshape(case["batch"], hk, -1, 1))
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = p * (torch.matmul(do, v.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)) / math.sqrt(case["dim"])
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q)
    t = s["q"].dtype
    return (_by_token(dq, case["q_len"], case["heads"]).to(t), _by_token(dk, case["kv_len"], hk).to(t),
            _by_token(dv, case["kv_len"], hk).to(t))


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    rstd = (((x - mean) ** 2).mean(1, keepdim=True) + EPS).rsqrt()
    y = (x - mean) * rstd * s["gamma"].float() + s["beta"].float()
    return y.to(s["x"].dtype), mean[:, 0], rstd[:, 0]


def _plain_norm_backward(s):
    dy, g = s["dout"].float(), s["gamma"]
    hat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    w = dy * g.float()
    dx = (w - w.mean(1, keepdim=True) - hat * (w * hat).mean(1, keepdim=True)) * s["rstd"][:, None]
    return dx.to(s["x"].dtype), (dy * hat).sum(0).to(g.dtype), dy.sum(0).to(g.dtype)


# ---- the framework's calls ------------------------------------------------------------------
def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lightining-core_b200", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    import lightning_core_b200 as lc
    return lc


def _own_norm(lc, s):
    case, x = s["case"], s["x"]
    rows, cols = x.shape
    dt, pt = (lc.BF16 if case[n] == "bf16" else lc.F32 for n in ("dtype", "params"))
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "norm_fwd":
        out = torch.empty_like(x)
        mean, rstd = torch.empty((2, rows), device="cuda")
        lc.check(lc.lib.lcLayerNormForward(x.data_ptr(), s["gamma"].data_ptr(), s["beta"].data_ptr(), out.data_ptr(),
                                           mean.data_ptr(), rstd.data_ptr(), rows, cols, 0, 0, EPS, dt, pt, stream))
        return out, mean, rstd
    dx = torch.empty_like(x)
    dgamma, dbeta = torch.empty_like(s["gamma"]), torch.empty_like(s["gamma"])
    lc.check(lc.lib.lcLayerNormBackward(s["dout"].data_ptr(), x.data_ptr(), s["gamma"].data_ptr(),
                                        s["mean"].data_ptr(), s["rstd"].data_ptr(), dx.data_ptr(), dgamma.data_ptr(),
                                        dbeta.data_ptr(), rows, cols, 0, 0, 0, dt, pt, stream))
    return dx, dgamma, dbeta


def _own_cross(lc, s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    by_q = (case["q_len"] * heads * dim, dim, heads * dim)  # batch, head and token strides
    by_k = (case["kv_len"] * kv_heads * dim, dim, kv_heads * dim)
    desc = lc.cross_attention_desc(case["batch"], heads, kv_heads, case["q_len"], case["kv_len"], dim,
                                   lc.BF16 if case["dtype"] == "bf16" else lc.F32, by_q, by_k, by_k, by_q,
                                   kv_lens=s["lens"].data_ptr() if s["lens"] is not None else None,
                                   key_mask=s["mask"].data_ptr() if s["mask"] is not None else None)
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "cross_bwd":
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        lc.check(lc.lib.lcCrossAttentionBackward(desc, s["dout"].data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                 s["out"].data_ptr(), s["lse"].data_ptr(), dq.data_ptr(),
                                                 dk.data_ptr(), dv.data_ptr(), stream))
        return dq, dk, dv
    out = torch.empty_like(q)
    lse = torch.empty((case["batch"], heads, case["q_len"]), device="cuda") if case["op"] == "cross_fwd" else None
    lc.check(lc.lib.lcCrossAttentionForward(desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                            lse.data_ptr() if lse is not None else None, None, stream))
    return (out, lse) if lse is not None else out


def run(state):
    op = state["case"]["op"]
    if own:
        return (_own_norm if op.startswith("norm") else _own_cross)(_framework(), state)
    if op == "norm_fwd":
        return _plain_norm(state)
    if op == "norm_bwd":
        return _plain_norm_backward(state)
    if op == "cross_bwd":
        return _plain_backward(state)
    out, lse = _plain_forward(state)
    return out if op == "cross_step" else (out, lse)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"].startswith("norm"):
        rows, cols, params = case["rows"], case["cols"], 2 if case["params"] == "bf16" else 4
        if case["op"] == "norm_fwd":  # x in, y out; gamma, beta in; mean, rstd out
            return {"bytes": 2 * rows * cols * size + 2 * cols * params + 8 * rows, "flops": 8 * rows * cols}
        # x and dy in, dx out; gamma in, two gradients out; mean, rstd in
        return {"bytes": 3 * rows * cols * size + 3 * cols * params + 8 * rows, "flops": 14 * rows * cols}
    seen, d = _keys_seen(case), case["dim"]
    of_q = case["batch"] * case["q_len"] * case["heads"] * d * size
    of_k = seen * case["kv_heads"] * d * size
    rows = 4 * case["batch"] * case["q_len"] * case["heads"]
    choice = {"all": 0, "lens": 4 * case["batch"], "mask": case["batch"] * case["kv_len"]}[case["keys"]]
    product = 2 * seen * case["q_len"] * case["heads"] * d
    if case["op"] == "cross_bwd":  # q, out, dout, k, v and the row sums in; three gradients out; five products
        grads = 2 * case["batch"] * case["kv_len"] * case["kv_heads"] * d * size
        return {"bytes": 4 * of_q + 2 * of_k + grads + rows + choice, "flops": 5 * product}
    kept = rows if case["op"] == "cross_fwd" else 0
    return {"bytes": 2 * of_q + 2 * of_k + kept + choice, "flops": 2 * product}


# ---- definitions in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = 1 / torch.sqrt(var + EPS)
        y = torch.addcmul(s["beta"].double(), (x - mean[:, None]) / torch.sqrt(var + EPS)[:, None], s["gamma"].double())
        return y, mean, rstd
    if case["op"] == "norm_bwd":
        # dx_j = sum_i w_i * d xhat_i / d x_j, with xhat = (x - mean) * rstd and w = gamma * dy
        dy, r = s["dout"].double(), s["rstd"].double()[:, None]
        hat = (s["x"].double() - s["mean"].double()[:, None]) * r
        w = dy * s["gamma"].double()
        n = case["cols"]
        dx = r / n * (n * w - w.sum(1, keepdim=True) - hat * torch.einsum("rc,rc->r", w, hat)[:, None])
        return dx, torch.einsum("rc,rc->c", dy, hat), torch.einsum("rc->c", dy)
    group = case["heads"] // case["kv_heads"]
    parts = []
    for b in range(case["batch"]):
        at = torch.arange(case["kv_len"], device="cuda")
        if s["lens"] is not None:
            at = at[: int(s["lens"][b])]
        elif s["mask"] is not None:
            at = at[s["mask"][b] != 0]
        q, k, v = (s[n][b].double() for n in ("q", "k", "v"))
        k, v = (x[at].repeat_interleave(group, 1) for x in (k, v))
        a = torch.einsum("thd,nhd->htn", q, k) * case["dim"] ** -0.5
        if case["op"] != "cross_bwd":
            lse = torch.logsumexp(a, -1)
            parts.append((torch.einsum("htn,nhd->thd", torch.exp(a - lse[..., None]), v), lse))
            continue
        do, o = s["dout"][b].double(), s["out"][b].double()
        p = torch.exp(a - s["lse"][b].double()[..., None])
        da = p * (torch.einsum("thd,nhd->htn", do, v) - torch.einsum("thd,thd->ht", do, o)[..., None])
        da = da * case["dim"] ** -0.5
        dk = torch.zeros((case["kv_len"], case["kv_heads"], case["dim"]), dtype=torch.float64, device="cuda")
        dv = torch.zeros_like(dk)
        shape = (len(at), case["kv_heads"], group, case["dim"])
        dk[at] = torch.einsum("htn,thd->nhd", da, q).reshape(shape).sum(2)
        dv[at] = torch.einsum("htn,thd->nhd", p, do).reshape(shape).sum(2)
        parts.append((torch.einsum("htn,nhd->thd", da, k), dk, dv))
    whole = [torch.stack(x) for x in zip(*parts)]
    return whole[0] if case["op"] == "cross_step" else tuple(whole)
