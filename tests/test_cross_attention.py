"""lcCrossAttentionForward / lcCrossAttentionBackward: refusals on the CPU, values on a B200 against the
formulas in 64 bits.

Tolerances, element by element, with u = 2^-24 and r half a step of the tensors' type (bf16 2^-8,
fp32 u).  A score is a dot product of d terms: off by es = scale * (d + 4) u sum|q||k| at most.  A weight
p is then off by p * (2 es + ep), where ep is its own rounding: r (bf16 weights enter the second product
as bf16) plus the exponential's error (2^-13 with bf16 tensors: the weights are rounded to 2^-8 anyhow;
2^-21 with fp32).  A sum over n weighted rows adds n u.  Results are rounded to the type: r."""
import itertools

import numpy as np
import pytest

U = 2.0 ** -24


# ---------------------------------------------------------------- CPU: refusals
def _desc(lc, **kw):
    a = dict(batch=2, q_heads=4, kv_heads=2, q_len=5, kv_len=7, head_dim=16, dtype=0)
    a.update(kw)
    return lc.cross_attention_desc(**a)


def _fwd(lc, desc, q=64, k=64, v=64, out=64, policy=None):
    return lc.lib.lcCrossAttentionForward(desc, q, k, v, out, None, policy, None)


def _bwd(lc, desc, dout=64, q=64, k=64, v=64, out=64, lse=64, dq=64, dk=64, dv=64):
    return lc.lib.lcCrossAttentionBackward(desc, dout, q, k, v, out, lse, dq, dk, dv, None)


INVALID = [dict(batch=0), dict(q_heads=0), dict(kv_heads=0), dict(q_len=0), dict(kv_len=0), dict(head_dim=0),
           dict(q_heads=5), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
           dict(out=(0, 16, 64)),        # two batch entries share memory
           dict(out=(320, 8, 64)),       # heads overlap
           dict(out=(320, 80, 15)),      # tokens overlap
           dict(k=(2 ** 59, 1, 1)), dict(batch=2 ** 20, q_heads=2 ** 10, kv_heads=2 ** 10, kv_len=2 ** 30)]
UNSUPPORTED = [dict(dtype=2), dict(dtype=9), dict(head_dim=257), dict(q_len=2 ** 31), dict(kv_len=2 ** 31 - 1),
               dict(batch=2 ** 31), dict(q_heads=2 ** 20, kv_heads=1, q_len=2 ** 12)]


@pytest.mark.parametrize("bad", INVALID)
def test_refuses_invalid(lc, bad):
    assert _fwd(lc, _desc(lc, **bad)) == lc.LC_INVALID_VALUE
    assert _bwd(lc, _desc(lc, **bad)) == lc.LC_INVALID_VALUE


@pytest.mark.parametrize("bad", UNSUPPORTED)
def test_refuses_unsupported(lc, bad):
    assert _fwd(lc, _desc(lc, **bad)) == lc.LC_NOT_SUPPORTED
    assert _bwd(lc, _desc(lc, **bad)) == lc.LC_NOT_SUPPORTED


def test_refuses_null_pointers(lc):
    d = _desc(lc)
    assert lc.lib.lcCrossAttentionForward(None, 64, 64, 64, 64, None, None, None) == lc.LC_INVALID_VALUE
    for n in ("q", "k", "v", "out"):
        assert _fwd(lc, d, **{n: None}) == lc.LC_INVALID_VALUE
    for n in ("dout", "q", "k", "v", "out", "lse", "dk", "dv"):
        assert _bwd(lc, d, **{n: None}) == lc.LC_INVALID_VALUE
    assert _bwd(lc, d, dq=None, dk=None, dv=None) == lc.LC_INVALID_VALUE


def test_refuses_gradients_that_share_memory(lc):
    wide = (5 * 4 * 16, 16, 4 * 16)
    assert _bwd(lc, _desc(lc, q=(0, 16, 64))) == lc.LC_INVALID_VALUE             # one q for every batch entry
    assert _bwd(lc, _desc(lc, q=wide, k=(0, 16, 32))) == lc.LC_INVALID_VALUE     # k is shared, v is not
    assert _bwd(lc, _desc(lc, k=(224, 0, 16), v=(224, 0, 16))) == lc.LC_INVALID_VALUE  # key heads share memory


def test_refuses_host_tensors_with_strides_and_postprocess(lc):
    p = lc.default_attention_policy()
    for n in ("q", "k", "v", "out"):
        assert _fwd(lc, _desc(lc, **{n: (1000, 16, 64)}), policy=p) == lc.LC_NOT_SUPPORTED
    p.output_scale = 0.5
    assert _fwd(lc, _desc(lc), policy=p) == lc.LC_NOT_SUPPORTED


def test_python_checks(lc):
    z = np.zeros
    with pytest.raises(ValueError):
        lc.cross_attention(z((1, 3, 2, 8)), z((1, 2, 4, 8)), z((1, 2, 4, 8)))
    with pytest.raises(ValueError):
        lc.cross_attention(z((1, 2, 2, 8)), z((1, 2, 4, 8)), z((1, 2, 5, 8)))
    with pytest.raises(ValueError):
        lc.cross_attention(z((1, 2, 2, 8)), z((1, 2, 4, 8)), z((1, 2, 4, 8)), kv_lens=[1, 2])
    with pytest.raises(ValueError):
        lc.cross_attention(z((1, 2, 2, 8)), z((1, 2, 4, 8)), z((1, 2, 4, 8)), key_mask=z((1, 5)))
    with pytest.raises(ValueError):
        lc.cross_attention(z((1, 2, 2, 8)), z((1, 2, 4, 8)), z((1, 2, 4, 8)), dtype=lc.BF16)


# ---------------------------------------------------------------- GPU
HOLE = 7.0  # what memory that must stay untouched holds


class Case:
    """Tensors of one problem on the GPU, in a layout, with NaN wherever a mask hides something."""

    def __init__(self, torch, lc, b, hq, hk, nq, nk, d, dtype="f32", keys="all", queries="all", layout="dense", seed=0,
                 scale=0.0, shared=False, spread=1.0):
        self.torch, self.lc = torch, lc
        self.b, self.hq, self.hk, self.nq, self.nk, self.d = b, hq, hk, nq, nk, d
        self.t = torch.bfloat16 if dtype == "bf16" else torch.float32
        self.r = 2.0 ** -8 if dtype == "bf16" else U
        self.ep = self.r + (2.0 ** -13 if dtype == "bf16" else 2.0 ** -21)
        self.scale = scale or d ** -0.5
        self.layout, self.shared = layout, shared
        g = torch.Generator(device="cuda").manual_seed(seed + 1000 * nq + nk)
        rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
        self.kv_lens = self.q_lens = self.key_mask = None
        vis = torch.ones((b, nk), dtype=torch.bool, device="cuda")
        rows = torch.ones((b, nq), dtype=torch.bool, device="cuda")
        if keys in ("lens", "both"):
            lens = torch.tensor([(0, nk, 1, nk // 2, nk + 9, -3, nk - 1, 65)[(i + 1 if b > 1 else 3) % 8]
                                 for i in range(b)], dtype=torch.int32, device="cuda")
            self.kv_lens = lens
            vis &= torch.arange(nk, device="cuda")[None] < lens[:, None]
        if keys in ("mask", "both"):
            m = torch.rand((b, nk), generator=g, device="cuda") < 0.6
            m[b // 2] = b == 1 or False  # one batch entry without a key (several, where there are more)
            m[:, nk // 3: nk // 3 + 130] &= nk < 300  # a whole tile hidden
            self.key_mask = (m.to(torch.uint8) * 255)
            vis &= m
        if queries == "lens":
            self.q_lens = torch.tensor([(nq // 2, nq, 0, nq + 5, 1, -1)[i % 6] for i in range(b)], dtype=torch.int32,
                                       device="cuda")
            rows &= torch.arange(nq, device="cuda")[None] < self.q_lens[:, None]
        self.vis, self.rows = vis, rows
        kb = 1 if shared else b
        self.q, self.qs = self.place(rnd(b, hq, nq, d) * spread)
        self.k, self.ks = self.place(rnd(kb, hk, nk, d))
        self.v, self.vs = self.place(rnd(kb, hk, nk, d))
        self.dout, self.os = self.place(rnd(b, hq, nq, d))
        # Hidden keys, values and rows hold NaN and infinities (a shared key only where all hide it).
        hide = ~(vis.any(0, keepdim=True) if shared else vis)
        self.k.masked_fill_(hide[:, None, :, None], float("nan"))
        self.v.masked_fill_(hide[:, None, :, None], float("inf"))
        self.q.masked_fill_(~rows[:, None, :, None], float("nan"))
        self.dout.masked_fill_(~rows[:, None, :, None], float("nan"))
        if shared:
            self.ks = (0,) + self.ks[1:]
            self.vs = (0,) + self.vs[1:]

    def place(self, x):
        """x [b, h, n, d] in memory of the layout; returns the view and its strides."""
        torch = self.torch
        b, h, n, d = x.shape
        if self.layout == "dense":
            s, size = (h * n * d, n * d, d), b * h * n * d
        elif self.layout == "tokens":   # [b, n, h, d]
            s, size = (n * h * d, d, h * d), b * h * n * d
        elif self.layout == "packed":   # a slice of [b, n, 3, h, d]
            s, size = (n * 3 * h * d, d, 3 * h * d), b * n * 3 * h * d
        else:                           # "odd": no alignment anywhere
            s = (h * (n * (d + 1) + 3) + 5, n * (d + 1) + 3, d + 1)
            size = b * s[0]
        buf = torch.full((size + 1,), HOLE, device="cuda", dtype=self.t)
        off = 1 if self.layout == "odd" else 0
        view = torch.as_strided(buf, (b, h, n, d), s + (1,), off)
        view.copy_(x.to(self.t))
        return view, s

    def like(self, x):
        """Memory of x's layout full of HOLE, and the view."""
        torch = self.torch
        base = torch.full((x.untyped_storage().nbytes() // x.element_size(),), HOLE, device="cuda", dtype=self.t)
        return base, torch.as_strided(base, x.shape, x.stride(), x.storage_offset())

    def desc(self):
        p = lambda t: t.data_ptr() if t is not None else None
        return self.lc.cross_attention_desc(self.b, self.hq, self.hk, self.nq, self.nk, self.d,
                                            self.lc.BF16 if self.r != U else self.lc.F32, self.qs, self.ks, self.vs,
                                            self.os, p(self.q_lens), p(self.kv_lens), p(self.key_mask), self.scale)

    def after_fills(self, stream):
        """A stream of the caller's waits for what was written on torch's."""
        cur = self.torch.cuda.current_stream()
        if stream is not None and stream != cur.cuda_stream:
            self.torch.cuda.ExternalStream(stream).wait_stream(cur)

    def forward(self, stream=None, want_lse=True):
        torch = self.torch
        self.out_mem, self.out = self.like(self.dout)
        self.lse = torch.full((self.b, self.hq, self.nq), HOLE, device="cuda")
        self.after_fills(stream)
        self.lc.check(self.lc.lib.lcCrossAttentionForward(self.desc(), self.q.data_ptr(), self.k.data_ptr(),
                                                          self.v.data_ptr(), self.out.data_ptr(),
                                                          self.lse.data_ptr() if want_lse else None, None, stream))
        return self.out, self.lse

    def backward(self, out, lse, dq=True, dkv=True, stream=None):
        self.mem, grads = zip(*(self.like(x) for x in (self.q, self.k, self.v)))
        p = [g.data_ptr() for g in grads]
        self.after_fills(stream)
        self.lc.check(self.lc.lib.lcCrossAttentionBackward(
            self.desc(), self.dout.data_ptr(), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), out.data_ptr(),
            lse.data_ptr(), p[0] if dq else None, p[1] if dkv else None, p[2] if dkv else None, stream))
        return grads

    def wide(self):
        """64-bit operands by query head, hidden values 0."""
        b, hq, hk = self.b, self.hq, self.hk
        by = lambda x: x.double().nan_to_num(0, 0, 0).expand(b, -1, -1, -1).repeat_interleave(hq // hk, 1)
        q = self.q.double().nan_to_num(0)
        return q, by(self.k), by(self.v)

    def scores(self):
        torch = self.torch
        q, k, _ = self.wide()
        s = torch.where(self.vis[:, None, None, :], q @ k.transpose(-1, -2) * self.scale, -float("inf"))
        # the scale is an fp32 number on the GPU: u more
        es = self.scale * (self.d + 5) * U * (q.abs() @ k.abs().transpose(-1, -2)) + 4 * U * s.abs().nan_to_num(0, 0, 0)
        return s, es

    def check_forward(self):
        torch = self.torch
        s, es = self.scores()
        _, _, v = self.wide()
        lse = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[..., None]).nan_to_num(0)  # rows without a key
        want = p @ v
        worst = torch.where(self.vis[:, None, None, :], es, 0).amax(-1, keepdim=True)
        n = self.nk
        tol = (p @ v.abs()) * (4 * worst + self.ep + self.ep + (n + 8) * U) + 2 * self.r * want.abs()
        rows = self.rows[:, None, :, None].expand_as(want)
        err = (self.out.double() - want).abs()
        bad = rows & ~(err <= tol + 1e-30)
        assert not bool(bad.any()), (int(bad.sum()), float((err / (tol + 1e-30))[rows].max()))
        ok = torch.isinf(lse) | ((self.lse.double() - lse).abs() <= 2 * worst[..., 0] + self.ep + (n + 4) * U +
                                 4 * U * lse.abs())
        ok &= ~torch.isinf(lse) | (self.lse == -float("inf"))
        assert bool((ok | ~self.rows[:, None, :]).all())
        # Rows past q_lens and everything between the rows hold what they held.
        assert bool((self.out.float()[~rows] == HOLE).all()) and bool((self.lse[~self.rows[:, None, :].expand_as(
            self.lse)] == HOLE).all())
        self.holes(self.out_mem, self.out)

    def holes(self, mem, view):
        torch = self.torch
        gap = torch.ones_like(mem, dtype=torch.bool)
        torch.as_strided(gap, view.shape, view.stride(), view.storage_offset()).fill_(False)
        assert bool((mem[gap].float() == HOLE).all())

    def check_backward(self, out, lse, grads):
        torch = self.torch
        q, k, v = self.wide()
        rows = self.rows[:, None, :, None]
        do = torch.where(rows, self.dout.double(), 0)
        o = torch.where(rows, out.double(), 0)
        s, es = self.scores()
        l = torch.where(torch.isinf(lse), float("inf"), lse.double())[..., None]
        p = torch.where(rows, torch.exp(s - torch.where(rows, l, float("inf"))), 0)
        rp = 2 * es + 2 * self.ep + 4 * U * l.abs().nan_to_num(0, 0, 0)  # relative error of a weight
        rp = torch.where(self.vis[:, None, None, :], rp, 0)
        dp, dd = do @ v.transpose(-1, -2), (do * o).sum(-1, keepdim=True)
        ds = p * (dp - dd)
        eds = ds.abs() * (rp + self.ep) + p * (self.d + 4) * U * (do.abs() @ v.abs().transpose(-1, -2) +
                                                              (do * o).abs().sum(-1, keepdim=True))
        n = max(self.nk, self.nq * self.hq // self.hk * (self.b if self.shared else 1))

        def by_key(x):  # sums over the heads of a key head, and over the batch when it is shared
            x = x.reshape(self.b, self.hk, self.hq // self.hk, self.nk, self.d).sum(2)
            return x.sum(0, keepdim=True) if self.shared else x

        want = [self.scale * ds @ k, by_key(self.scale * ds.transpose(-1, -2) @ q), by_key(p.transpose(-1, -2) @ do)]
        tol = [self.scale * (eds @ k.abs() + (n + 8) * U * (ds.abs() @ k.abs())),
               by_key(self.scale * (eds.transpose(-1, -2) @ q.abs() + (n + 8) * U * (ds.abs().transpose(-1, -2) @ q.abs()))),
               by_key((p * (rp + (n + 8) * U)).transpose(-1, -2) @ do.abs())]
        for i, name in enumerate(("dq", "dk", "dv")):
            live = rows.expand_as(want[0]) if i == 0 else torch.ones_like(want[i], dtype=torch.bool)
            t = tol[i] + 2 * self.r * want[i].abs() + 1e-30
            err = (grads[i].double() - want[i]).abs()
            bad = live & ~(err <= t)
            assert not bool(bad.any()), (name, int(bad.sum()), float((err / t)[live].max()))
            assert bool((grads[i].float()[~live] == HOLE).all())
            self.holes(self.mem[i], grads[i])


def _both(torch, lc, *a, **kw):
    c = Case(torch, lc, *a, **kw)
    out, lse = c.forward()
    torch.cuda.synchronize()
    c.check_forward()
    out, lse = out.clone(memory_format=torch.preserve_format), lse.clone()
    # clone() need not keep a view's gaps: the call wants out laid out as dout
    mem, o = c.like(c.dout)
    o.copy_(out)
    grads = c.backward(o, lse)
    torch.cuda.synchronize()
    c.check_backward(o, lse, grads)
    return c, o, lse, grads


# batch, q_heads, kv_heads, q_len, kv_len, head_dim
SIZES = [(1, 1, 1, 1, 1, 1), (1, 2, 1, 3, 2, 5), (2, 2, 2, 1, 17, 64), (3, 4, 2, 5, 63, 64), (1, 3, 3, 64, 64, 32),
         (2, 6, 2, 33, 65, 128), (4, 2, 1, 17, 129, 80), (2, 2, 2, 130, 300, 64), (5, 4, 4, 65, 127, 128),
         (2, 8, 1, 1, 700, 128), (1, 2, 2, 2, 1025, 96), (2, 2, 1, 9, 70, 200), (1, 1, 1, 40, 257, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("keys,queries,layout", [("all", "all", "dense"), ("lens", "all", "tokens"),
                                                 ("mask", "lens", "packed"), ("both", "lens", "odd")])
def test_small(gpu, size, dtype, keys, queries, layout):
    import torch
    _both(torch, gpu, *size, dtype=dtype, keys=keys, queries=queries, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("keys", ["all", "lens", "mask"])
@pytest.mark.parametrize("size", [(2, 4, 4, 128, 128, 64), (2, 4, 2, 200, 384, 128), (3, 4, 1, 257, 513, 64),
                                  (1, 2, 2, 300, 1100, 128), (2, 2, 2, 700, 90, 64), (6, 2, 2, 127, 255, 128)])
def test_tiles(gpu, size, dtype, keys):
    """Whole and ragged tiles of 128 rows and keys, with shared heads and hidden tiles."""
    import torch
    _both(torch, gpu, *size, dtype=dtype, keys=keys, queries="lens" if keys == "lens" else "all", layout="tokens")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(3, 2, 2, 40, 100, 64), (4, 4, 2, 1, 300, 128), (3, 4, 2, 150, 200, 128), (2, 2, 1, 5, 9, 24)])
@pytest.mark.parametrize("keys", ["all", "lens", "mask"])
def test_source_shared_by_the_batch(gpu, size, dtype, keys):
    """One source for every batch entry: its gradient is the sum over them."""
    import torch
    _both(torch, gpu, *size, dtype=dtype, keys=keys, layout="tokens", shared=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq", [1, 3, 200])
def test_large_scores(gpu, dtype, nq):
    """Scores up to a few hundred: one key takes nearly all the weight, the row maximum moves."""
    import torch
    c = Case(torch, gpu, 2, 4, 2, nq, 600, 64, dtype=dtype, layout="tokens", spread=20.0)
    c.forward()
    torch.cuda.synchronize()
    c.check_forward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("f32", 64), ("bf16", 64), ("bf16", 128), ("bf16", 40)])
def test_each_gradient_alone_and_again(gpu, dtype, d):
    """dq alone, dk and dv alone, and the same bits in every call, forward too."""
    import torch
    c, o, lse, grads = _both(torch, gpu, 2, 4, 2, 150, 333, d, dtype=dtype, keys="lens", layout="tokens")
    for _ in range(3):
        again = c.backward(o, lse)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, grads))
    q_only = c.backward(o, lse, dkv=False)
    torch.cuda.synchronize()
    assert torch.equal(q_only[0], grads[0]) and bool((q_only[1].float() == HOLE).all())
    kv_only = c.backward(o, lse, dq=False)
    torch.cuda.synchronize()
    assert torch.equal(kv_only[1], grads[1]) and torch.equal(kv_only[2], grads[2])
    assert bool((kv_only[0].float() == HOLE).all())
    for _ in range(3):
        o2, l2 = c.forward()
        torch.cuda.synchronize()
        assert torch.equal(o2, o) and torch.equal(l2, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nk", [(1, 900), (4, 2000), (140, 300)])
def test_streams_and_graph(gpu, dtype, nq, nk):
    """Calls on two streams at once keep their own workspaces; a captured pair replays."""
    import torch
    c, o, lse, grads = _both(torch, gpu, 2, 4, 4, nq, nk, 64, dtype=dtype, keys="mask", layout="tokens")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs, gs = [], []
    for i in range(8):
        outs.append(c.forward(streams[i % 2].cuda_stream))
        gs.append(c.backward(o, lse, stream=streams[i % 2].cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) and torch.equal(b, lse) for a, b in outs)
    assert all(torch.equal(a, b) for g in gs for a, b in zip(g, grads))
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        s = torch.cuda.current_stream().cuda_stream
        o2, l2 = c.forward(s)
        g2 = c.backward(o2, l2, stream=s)
    for _ in range(3):
        o2.zero_()
        gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(o2, o) and torch.equal(l2, lse) and all(torch.equal(a, b) for a, b in zip(g2, grads))


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """The backward pass against central differences of the definition in 64-bit arithmetic."""
    rng = np.random.default_rng(4)
    b, hq, hk, nq, nk, d, h = 2, 2, 1, 3, 5, 4, 1e-5
    x = [rng.standard_normal(s) for s in ((b, hq, nq, d), (b, hk, nk, d), (b, hk, nk, d))]
    dout = rng.standard_normal((b, hq, nq, d))
    lens = np.array([5, 3])

    def loss(q, k, v):
        k, v = np.repeat(k, hq // hk, 1), np.repeat(v, hq // hk, 1)
        s = q @ k.swapaxes(-1, -2) / np.sqrt(d)
        s = np.where(np.arange(nk)[None, None, None] < lens[:, None, None, None], s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        return float(((p / p.sum(-1, keepdims=True)) @ v * dout).sum())

    out, lse = gpu.cross_attention(*x, kv_lens=lens)
    got = gpu.cross_attention_backward(dout, *x, out, lse, kv_lens=lens)
    for i in range(3):
        want = np.zeros_like(x[i])
        for at in np.ndindex(*x[i].shape):
            up, down = [t.copy() for t in x], [t.copy() for t in x]
            up[i][at] += h
            down[i][at] -= h
            want[at] = (loss(*up) - loss(*down)) / (2 * h)
        np.testing.assert_allclose(got[i], want, atol=2e-5, rtol=1e-5)


@pytest.mark.gpu
def test_host_arrays(gpu):
    """The Python call on host arrays: the policy's uploads and downloads, rows past q_lens as they were."""
    lc = gpu
    rng = np.random.default_rng(8)
    q, k, v = (rng.standard_normal(s).astype(np.float32) for s in ((2, 4, 6, 32), (2, 2, 50, 32), (2, 2, 50, 32)))
    mask = rng.random((2, 50)) < 0.7
    out, lse = lc.cross_attention(q, k, v, kv_lens=[50, 20], key_mask=mask, q_lens=[6, 2])
    assert not out[1, :, 2:].any() and not lse[1, :, 2:].any()
    vis = mask & (np.arange(50)[None] < np.array([50, 20])[:, None])
    kk, vv = np.repeat(k, 2, 1).astype(np.float64), np.repeat(v, 2, 1).astype(np.float64)
    s = np.where(vis[:, None, None], q @ kk.swapaxes(-1, -2) / np.sqrt(32), -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    want = p / p.sum(-1, keepdims=True) @ vv
    want[1, :, 2:] = 0
    # scores of 32 terms of order 1: 37 u of their absolute sum (below 20), twice, and 50 u more
    np.testing.assert_allclose(out, want, atol=2 * (2 * 37 * 20 * 32 ** -0.5 + 50) * U * 3)
    b_out, _ = lc.cross_attention(lc.to_bf16(q), lc.to_bf16(k), lc.to_bf16(v), kv_lens=[50, 20], key_mask=mask,
                                  q_lens=[6, 2], dtype=lc.BF16)
    np.testing.assert_allclose(lc.from_bf16(b_out), want, atol=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,nq", [("bf16", 64, 70), ("bf16", 128, 70), ("bf16", 64, 1), ("f32", 64, 70), ("f32", 128, 3)])
@pytest.mark.parametrize("nk", [1, 2, 5, 33])
def test_log_sum_of_few_keys(gpu, dtype, d, nq, nk):
    """lse with scores that are exact in any order (entries -1, 0, 1): what is left is the scale's and the
    subtraction's rounding (|s| < 16 * log2 e: 2 * 2^-24 * 24), the exponential (2.7e-6), the sum (n u) and the
    logarithm (2^-22 of a result below 8)."""
    import torch
    lc = gpu
    g = torch.Generator(device="cuda").manual_seed(nk + nq)
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    pick = lambda *s: torch.randint(-1, 2, s, generator=g, device="cuda").to(t)
    q, k, v = pick(2, 4, nq, d), pick(2, 2, nk, d), pick(2, 2, nk, d)
    out, lse = torch.empty_like(q), torch.empty((2, 4, nq), device="cuda")
    desc = lc.cross_attention_desc(2, 4, 2, nq, nk, d, lc.BF16 if dtype == "bf16" else lc.F32)
    lc.check(lc.lib.lcCrossAttentionForward(desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                                            None, None))
    s = torch.einsum("bhtd,bhnd->bhtn", q.double(), k.double().repeat_interleave(2, 1)) * d ** -0.5
    assert s.abs().max() < 16
    torch.cuda.synchronize()
    off = (lse.double() - torch.logsumexp(s, -1)).abs().max().item()
    assert off <= 48 * U + 2.7e-6 + nk * U + 8 * 4 * U


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 13000, 64), (1, 1, 1, 1, 9000, 128), (1, 1, 1, 17, 3000, 64),
                                  (1, 1, 1, 33, 1500, 128), (1, 3, 1, 1, 5000, 128), (1, 1, 1, 9, 2500, 200)])
def test_odd_rows_split_over_the_keys(gpu, size, dtype):
    """An odd number of rows in an odd number of parts: the parts' statistics and sums share a workspace."""
    import torch
    _both(torch, gpu, *size, dtype=dtype, keys="mask")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 44])
@pytest.mark.parametrize("hq,nq", [(2, 1), (4, 1), (3, 1), (2, 4), (2, 5), (2, 8), (16, 1), (17, 1)])
def test_row_counts_where_the_kernel_changes(gpu, dtype, d, hq, nq):
    import torch
    _both(torch, gpu, 3, hq, 1, nq, 190, d, dtype=dtype, keys="lens", queries="lens", layout="tokens")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,stride", [("bf16", 2 ** 32 + 64), ("f32", 2 ** 31 + 64)])
@pytest.mark.parametrize("nq", [1, 40])
@pytest.mark.parametrize("d", [64, 72])
def test_offsets_past_32_bits(gpu, dtype, stride, nq, d):
    """Batch entries of k, v and their gradients further apart than 32 bits reach, against the same values dense."""
    import torch
    lc, t = gpu, torch.bfloat16 if dtype == "bf16" else torch.float32
    dt = lc.BF16 if dtype == "bf16" else lc.F32
    b, h, nk = 2, 2, 150
    g = torch.Generator(device="cuda").manual_seed(3)
    near = [torch.randn((b, h, n, d), generator=g, device="cuda").to(t) for n in (nq, nq, nk, nk)]
    q, do = near[:2]
    far = []
    for x in near[2:] + [near[2], near[3]]:
        y = torch.as_strided(torch.empty(stride + h * nk * d, device="cuda", dtype=t), (b, h, nk, d), (stride, nk * d, d, 1))
        y.copy_(x)
        far.append(y)
    got = []
    for k, v, dk, dv, s in ((near[2], near[3], near[2].clone(), near[3].clone(), (h * nk * d, nk * d, d)),
                            (*far, (stride, nk * d, d))):
        o, dq, lse = torch.empty_like(q), torch.empty_like(q), torch.empty((b, h, nq), device="cuda")
        desc = lc.cross_attention_desc(b, h, h, nq, nk, d, dt, k=s, v=s)
        lc.check(lc.lib.lcCrossAttentionForward(desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                                lse.data_ptr(), None, None))
        lc.check(lc.lib.lcCrossAttentionBackward(desc, do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                                 lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), None))
        torch.cuda.synchronize()
        got.append((o, lse, dq, dk, dv))
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nk,d", [(1, 5000, 64), (2, 700, 128), (70, 2000, 64), (300, 300, 128)])
def test_two_graphs_at_once(gpu, dtype, nq, nk, d):
    """Two captured calls replayed on two streams at once do not share their workspaces."""
    import torch
    lc = gpu
    cases, graphs, outs = [], [], []
    for seed in (1, 2):
        c, o, lse, grads = _both(torch, lc, 1, 2, 1, nq, nk, d, dtype=dtype, keys="mask", seed=seed)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            s = torch.cuda.current_stream().cuda_stream
            o2, l2 = c.forward(s)
            g2 = c.backward(o2, l2, stream=s)
        cases.append((o, lse, *grads))
        graphs.append(gr)
        outs.append((o2, l2, *g2))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for want, got in zip(cases, outs) for x, y in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_only_dq_with_a_shared_source(gpu, dtype, d):
    import torch
    c, o, lse, grads = _both(torch, gpu, 3, 4, 2, 30, 200, d, dtype=dtype, keys="lens", shared=True)
    again = c.backward(o, lse, dkv=False)
    torch.cuda.synchronize()
    # Another kernel may serve this call: in fp32 each is off by at most (200 + 8) * 2^-22 of sums of magnitudes,
    # which exceed the largest result by sqrt(200) or so.
    off = float((again[0].double() - grads[0].double()).abs().max())
    assert off <= (2 * 208 * 2.0 ** -22 * 15 * float(grads[0].double().abs().max()) if dtype == "f32" else 0.0)
    assert bool((again[1].float() == HOLE).all()) and bool((again[2].float() == HOLE).all())


def _block(torch, lc, x, mem, gamma, beta, w, dy, heads, lens, stream):
    """Norm, projections and cross attention over `mem` as a decoder layer uses them, and the way back; every
    tensor by token, [batch, tokens, columns].  Returns y and the gradients of x, gamma, beta, w and mem."""
    b, n, c = x.shape
    nk, d = mem.shape[1], c // heads
    L, new = lc.lib, lambda *s: torch.empty(s, device="cuda")

    def mm(a, bmat):
        out = new(a.shape[0], bmat.shape[1])
        lc.check(L.lcMatMul(a.data_ptr(), bmat.data_ptr(), out.data_ptr(), a.shape[0], a.shape[1], bmat.shape[1], lc.F32,
                            None, stream))
        return out

    xf, mf, dyf = x.reshape(b * n, c), mem.reshape(b * nk, c), dy.reshape(b * n, c)
    h, stats, lse = new(b * n, c), new(2, b * n), new(b, heads, n)
    lc.check(L.lcLayerNormForward(xf.data_ptr(), gamma.data_ptr(), beta.data_ptr(), h.data_ptr(), stats[0].data_ptr(),
                                  stats[1].data_ptr(), b * n, c, 0, 0, 1e-5, lc.F32, lc.F32, stream))
    q, kv = mm(h, w["q"]), mm(mf, w["kv"])
    k, v = kv, kv[:, c:]
    by_q, by_k = (n * c, d, c), (nk * 2 * c, d, 2 * c)
    desc = lc.cross_attention_desc(b, heads, heads, n, nk, d, lc.F32, by_q, by_k, by_k, by_q, kv_lens=lens.data_ptr())
    o, dq, dkv, dx = new(b * n, c), new(b * n, c), new(b * nk, 2 * c), new(b * n, c)
    lc.check(L.lcCrossAttentionForward(desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), None,
                                       stream))
    y = mm(o, w["o"])
    do = mm(dyf, w["o"].T.contiguous())
    lc.check(L.lcCrossAttentionBackward(desc, do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                        lse.data_ptr(), dq.data_ptr(), dkv.data_ptr(), dkv[:, c:].data_ptr(), stream))
    dh = mm(dq, w["q"].T.contiguous())
    dgamma, dbeta = new(c), new(c)
    lc.check(L.lcLayerNormBackward(dh.data_ptr(), xf.data_ptr(), gamma.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(),
                                   dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(), b * n, c, 0, 0, 0, lc.F32, lc.F32,
                                   stream))
    return [y, dx, dgamma, dbeta, mm(h.T.contiguous(), dq), mm(mf.T.contiguous(), dkv), mm(o.T.contiguous(), dyf),
            mm(dkv, w["kv"].T.contiguous())]


@pytest.mark.gpu
@pytest.mark.parametrize("n,nk,heads,c", [(1, 33, 2, 64), (19, 70, 4, 256), (130, 200, 2, 256)])
def test_a_decoder_layer(gpu, n, nk, heads, c):
    """The operators together, eager and captured, on a stream of their own, against 64-bit autograd.  Tolerance:
    seven stages one after the other, each off by at most (m + 8) * 2^-22 of its sums of magnitudes, m terms or fewer
    (2^-22: the split of the fp32 products); sums of magnitudes exceed the results' largest by sqrt(m) or so."""
    import torch
    lc, b = gpu, 2
    g = torch.Generator(device="cuda").manual_seed(n)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")
    x, mem, dy = rnd(b, n, c), rnd(b, nk, c), rnd(b, n, c)
    gamma, beta = 1 + 0.1 * rnd(c), 0.1 * rnd(c)
    w = {"q": rnd(c, c) * c ** -0.5, "kv": rnd(c, 2 * c) * c ** -0.5, "o": rnd(c, c) * c ** -0.5}
    lens = torch.tensor([nk, nk // 2 + 1], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _block(torch, lc, x, mem, gamma, beta, w, dy, heads, lens, side.cuda_stream)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        again = _block(torch, lc, x, mem, gamma, beta, w, dy, heads, lens, torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        for t in again:
            t.fill_(0)
        gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, again))

    leaves = [t.double().requires_grad_() for t in (x, gamma, beta, w["q"], w["kv"], w["o"], mem)]
    x_, gm, bt, wq, wkv, wo, mem_ = leaves
    h = torch.nn.functional.layer_norm(x_, (c,), gm, bt, 1e-5)
    heads_of = lambda t: t.unflatten(-1, (heads, -1)).transpose(1, 2)
    k, v = (mem_ @ wkv).chunk(2, -1)
    s = heads_of(h @ wq) @ heads_of(k).transpose(-1, -2) * (c // heads) ** -0.5
    hidden = torch.arange(nk, device="cuda")[None] >= lens[:, None]
    p = torch.softmax(s.masked_fill(hidden[:, None, None, :], -float("inf")), -1)
    y = (p @ heads_of(v)).transpose(1, 2).flatten(2) @ wo
    gx, ggm, gbt, gq, gkv, go, gmem = torch.autograd.grad(y, leaves, dy.double())
    want = [y, gx, ggm, gbt, gq, gkv, go, gmem]
    m = max(c, b * n, b * nk)
    for a, e in zip(got, want):
        e = e.detach().reshape(a.shape)
        assert float((a.double() - e).abs().max()) <= 7 * (m + 8) * 2.0 ** -22 * m ** 0.5 * float(e.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(4, 48, 3, 60, 180, 96), (4, 48, 3, 60, 180, 64), (4, 16, 1, 60, 600, 128)])
def test_rows_behind_a_sequence_never_reach_the_keys(gpu, size):
    """Many heads to a key head, each with a last tile whose rows behind q_lens hold NaN: the products with them
    wait for their zeroing, call after call."""
    import torch
    c, o, lse, grads = _both(torch, gpu, *size, dtype="bf16", keys="lens", queries="lens", layout="tokens")
    for _ in range(60):
        again = c.backward(o, lse)
        torch.cuda.synchronize()
        assert all(torch.equal(a.nan_to_num(1), b.nan_to_num(1)) for a, b in zip(again, grads))
