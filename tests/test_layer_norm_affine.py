"""lcLayerNormForward / lcLayerNormBackward: refusals on the CPU, values on a B200 against the formulas in
64 bits.

Tolerances, with u = 2^-24 (half an fp32 step) and r half a step of the output type (bf16 2^-8): a sum runs
over at most N = 48 sequential adds and lane steps for the row statistics of up to 16384 columns, so
mean is off by at most N u avg|x|, and a row's terms by N u of their absolute sum; the tests below
write this out for each result.  Nothing was fitted to outputs."""
import ctypes as C

import numpy as np
import pytest

U = 2.0 ** -24
N = 48
EPS = 1e-5


# ---------------------------------------------------------------- CPU: refusals
def _fwd(lc, **kw):
    a = dict(x=64, gamma=None, beta=None, out=64, mean=None, rstd=None, rows=4, cols=8, xs=0, os=0, eps=EPS, dt=0, pt=0)
    a.update(kw)
    return lc.lib.lcLayerNormForward(a["x"], a["gamma"], a["beta"], a["out"], a["mean"], a["rstd"], a["rows"], a["cols"],
                                     a["xs"], a["os"], a["eps"], a["dt"], a["pt"], None)


def _bwd(lc, **kw):
    a = dict(dout=64, x=64, gamma=None, mean=64, rstd=64, dx=64, dg=None, db=None, rows=4, cols=8, ds=0, xs=0, gs=0, dt=0,
             pt=0)
    a.update(kw)
    return lc.lib.lcLayerNormBackward(a["dout"], a["x"], a["gamma"], a["mean"], a["rstd"], a["dx"], a["dg"], a["db"],
                                      a["rows"], a["cols"], a["ds"], a["xs"], a["gs"], a["dt"], a["pt"], None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(out=None), dict(rows=0), dict(cols=0), dict(xs=7), dict(os=5),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(rows=2 ** 61, cols=16)])
def test_forward_refuses_invalid(lc, bad):
    assert _fwd(lc, **bad) == lc.LC_INVALID_VALUE


@pytest.mark.parametrize("bad", [dict(dt=2), dict(pt=2), dict(dt=7), dict(rows=1, cols=2 ** 31)])
def test_forward_refuses_unsupported(lc, bad):
    assert _fwd(lc, **bad) == lc.LC_NOT_SUPPORTED


@pytest.mark.parametrize("bad", [dict(dout=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(dx=None),
                                 dict(rows=0), dict(cols=0), dict(ds=7), dict(xs=7), dict(gs=7)])
def test_backward_refuses_invalid(lc, bad):
    assert _bwd(lc, **bad) == lc.LC_INVALID_VALUE


@pytest.mark.parametrize("bad", [dict(dt=2), dict(pt=2)])
def test_backward_refuses_unsupported(lc, bad):
    assert _bwd(lc, **bad) == lc.LC_NOT_SUPPORTED


def test_python_checks(lc):
    x = np.zeros((3, 8), np.float32)
    with pytest.raises(ValueError):
        lc.layer_norm_affine(x, gamma=np.ones(7))
    with pytest.raises(ValueError):
        lc.layer_norm_affine(x, dtype=lc.BF16)
    with pytest.raises(ValueError):
        lc.layer_norm_affine(np.zeros((0, 8), np.float32))
    with pytest.raises(ValueError):
        lc.layer_norm_backward(np.zeros((3, 7)), x, np.zeros(3), np.ones(3))
    with pytest.raises(ValueError):
        lc.layer_norm_backward(x, x, np.zeros(4), np.ones(3))


# ---------------------------------------------------------------- GPU
def _types(lc, torch, name):
    return (torch.bfloat16, lc.BF16, 2.0 ** -8) if name == "bf16" else (torch.float32, lc.F32, U)


def _rows(torch, g, rows, cols, stride, t):
    """[rows, cols] with a row stride inside a larger buffer whose gaps hold NaN."""
    buf = torch.full((rows * stride + 16,), float("nan"), device="cuda", dtype=t)
    x = torch.as_strided(buf, (rows, cols), (stride, 1))
    x.copy_((torch.randn((rows, cols), generator=g, device="cuda") * 2 + torch.randn((rows, 1), generator=g,
                                                                                     device="cuda")).to(t))
    return buf, x


SHAPES = [(1, 1), (3, 2), (5, 31), (8, 64), (7, 256), (9, 264), (2, 500), (33, 512), (40, 1000), (17, 1024), (6, 1333),
          (300, 1536), (4, 2047), (5, 4096), (3, 4104), (3, 8192), (2, 8191), (5, 9001), (3, 16384), (2, 20000)]


def _forward_check(torch, lc, x, gamma, beta, out, mean, rstd, r):
    x, gm = x.double(), (gamma.double() if gamma is not None else torch.ones((), device="cuda", dtype=torch.float64))
    bt = beta.double() if beta is not None else torch.zeros((), device="cuda", dtype=torch.float64)
    n = max(N, x.shape[1] / 1024 + 16)
    mu = x.mean(1, keepdim=True)
    var = ((x - mu) ** 2).mean(1, keepdim=True)
    rs = 1 / torch.sqrt(var + EPS)
    y = (x - mu) * rs * gm + bt
    dmu = n * U * x.abs().mean(1, keepdim=True)  # error of the mean
    # d var / var + eps: the sum's own error, and twice the mean's error against sqrt(var) (its first
    # order cancels; kept as a bound); half of it reaches rstd.
    drs = rs * ((n + 4) * U + 2 * (dmu * rs) ** 2 + 2 * U * dmu * rs)
    tol = gm.abs() * (rs * dmu + (x - mu).abs() * drs) + 4 * U * (y.abs() + bt.abs() + (x * rs * gm).abs()) + r * y.abs()
    assert bool(((out.double() - y).abs() <= tol + 1e-30).all()), ((out.double() - y).abs() / (tol + 1e-30)).max()
    if mean is not None:
        assert bool(((mean.double() - mu[:, 0]).abs() <= dmu[:, 0] + 2 * U * mu[:, 0].abs()).all())
        assert bool(((rstd.double() - rs[:, 0]).abs() <= drs[:, 0] + 4 * U * rs[:, 0]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype,params,pad", [("f32", "f32", 0), ("bf16", "f32", 0), ("bf16", "bf16", 3), ("f32", "bf16", 8),
                                              ("bf16", None, 8)])
def test_forward(gpu, rows, cols, dtype, params, pad):
    import torch
    lc = gpu
    t, dt, r = _types(lc, torch, dtype)
    pt, pdt, _ = _types(lc, torch, params or "f32")
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + cols)
    xb, x = _rows(torch, g, rows, cols, cols + pad, t)
    ob, out = _rows(torch, g, rows, cols, cols + 2 * pad, t)
    ob.fill_(7.0)
    gamma = (1 + torch.randn(cols, generator=g, device="cuda")).to(pt) if params else None
    beta = torch.randn(cols, generator=g, device="cuda").to(pt) if params else None
    mean, rstd = torch.full((2, rows + 1), 7.0, device="cuda")
    lc.check(lc.lib.lcLayerNormForward(x.data_ptr(), gamma.data_ptr() if params else None,
                                       beta.data_ptr() if params else None, out.data_ptr(), mean.data_ptr(),
                                       rstd.data_ptr(), rows, cols, cols + pad, cols + 2 * pad, EPS, dt, pdt, None))
    torch.cuda.synchronize()
    _forward_check(torch, lc, x, gamma, beta, out, mean[:rows], rstd[:rows], r)
    assert float(mean[rows]) == 7.0 and float(rstd[rows]) == 7.0
    gaps = torch.ones_like(ob, dtype=torch.bool)
    torch.as_strided(gaps, (rows, cols), (cols + 2 * pad, 1)).fill_(False)
    assert bool((ob[gaps] == 7.0).all())  # nothing between or behind the rows is written


def _backward_check(torch, dout, x, gamma, mean, rstd, dx, dg, db, r, rp, row_adds):
    dy, x = dout.double(), x.double()
    gm = gamma.double() if gamma is not None else torch.ones((), device="cuda", dtype=torch.float64)
    mu, rs = mean.double()[:, None], rstd.double()[:, None]
    n = max(N, x.shape[1] / 1024 + 16)
    h = (x - mu) * rs
    dh = 2 * U * h.abs()
    w = dy * gm
    if dx is not None:
        m1, m2 = w.mean(1, keepdim=True), (w * h).mean(1, keepdim=True)
        want = rs * (w - m1 - h * m2)
        e1 = n * U * w.abs().mean(1, keepdim=True)
        e2 = (n + 4) * U * (w * h).abs().mean(1, keepdim=True)
        tol = rs * (e1 + h.abs() * e2 + 6 * U * (w.abs() + m1.abs() + (h * m2).abs())) + r * want.abs()
        assert bool(((dx.double() - want).abs() <= tol + 1e-30).all())
    for got, terms in ((dg, dy * h), (db, dy)):
        if got is None:
            continue
        want = terms.sum(0)
        tol = (row_adds + 4) * U * terms.abs().sum(0) + rp * want.abs()
        assert bool(((got.double() - want).abs() <= tol + 1e-30).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES + [(2501, 64), (1203, 1333), (901, 4096), (700, 9001)])
@pytest.mark.parametrize("dtype,params,pad", [("f32", "f32", 0), ("bf16", "f32", 8), ("bf16", "bf16", 0), ("f32", None, 3)])
def test_backward(gpu, rows, cols, dtype, params, pad):
    import torch
    lc = gpu
    t, dt, r = _types(lc, torch, dtype)
    pt, pdt, rp = _types(lc, torch, params or "f32")
    g = torch.Generator(device="cuda").manual_seed(rows * 5 + cols)
    _, x = _rows(torch, g, rows, cols, cols + pad, t)
    _, dout = _rows(torch, g, rows, cols, cols + 2 * pad, t)
    db_, dx = _rows(torch, g, rows, cols, cols + 3 * pad, t)
    db_.fill_(7.0)
    gamma = (1 + torch.randn(cols, generator=g, device="cuda")).to(pt) if params else None
    mean = x.double().mean(1)
    rstd = (((x.double() - mean[:, None]) ** 2).mean(1) + EPS).rsqrt().float()
    mean = mean.float()
    dg, db = torch.full((2, cols), 7.0, device="cuda", dtype=pt)

    def call(dx_, dg_, db__):
        lc.check(lc.lib.lcLayerNormBackward(dout.data_ptr(), x.data_ptr(), gamma.data_ptr() if params else None,
                                            mean.data_ptr(), rstd.data_ptr(), dx_.data_ptr() if dx_ is not None else None,
                                            dg_.data_ptr() if dg_ is not None else None,
                                            db__.data_ptr() if db__ is not None else None, rows, cols, cols + 2 * pad,
                                            cols + pad, cols + 3 * pad, dt, pdt, None))
        torch.cuda.synchronize()

    call(dx, dg, db)
    # A column's sum passes through at most `rows` adds in a thread, then a block's and the last ones.
    _backward_check(torch, dout, x, gamma, mean, rstd, dx, dg, db, r, rp, min(rows, 400) + 64)
    gaps = torch.ones_like(db_, dtype=torch.bool)
    torch.as_strided(gaps, (rows, cols), (cols + 3 * pad, 1)).fill_(False)
    assert bool((db_[gaps] == 7.0).all())
    # Each gradient alone, and the same bits again.
    dx2, dg2, db2 = torch.empty_like(db_), torch.empty_like(dg), torch.empty_like(db)
    dx2 = torch.as_strided(dx2, (rows, cols), (cols + 3 * pad, 1))
    call(dx2, None, None)
    call(None, dg2, None)
    call(None, None, db2)
    assert torch.equal(dx2, dx) and torch.equal(dg2, dg) and torch.equal(db2, db)


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """The backward pass against central differences of the forward pass in 64-bit arithmetic."""
    rng = np.random.default_rng(3)
    rows, cols, h = 5, 37, 1e-5
    x, dout, gamma, beta = (rng.standard_normal(s) for s in ((rows, cols), (rows, cols), cols, cols))

    def loss(x, gamma, beta):
        mu = x.mean(1, keepdims=True)
        y = (x - mu) / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + EPS) * gamma + beta
        return float((y * dout).sum())

    def diff(args, i):
        out = np.zeros_like(args[i])
        for at in np.ndindex(*args[i].shape):
            a, b = [t.copy() for t in args], [t.copy() for t in args]
            a[i][at] += h
            b[i][at] -= h
            out[at] = (loss(*a) - loss(*b)) / (2 * h)
        return out

    _, mean, rstd = gpu.layer_norm_affine(x, gamma, beta)
    got = gpu.layer_norm_backward(dout, x, mean, rstd, gamma)
    for i in range(3):
        # differences: h^2 of the third derivative (order 1) and 2^-53 of the loss (below 100) over h;
        # the kernel: fp32 inputs and sums of 37 terms of order 10
        np.testing.assert_allclose(got[i], diff((x, gamma, beta), i), atol=3e-5, rtol=1e-5)


@pytest.mark.gpu
def test_in_place_streams_graph_and_order(gpu):
    """out over x, dx over dout; two streams at once; a captured and replayed pair of calls."""
    import torch
    lc = gpu
    g = torch.Generator(device="cuda").manual_seed(1)
    for cols in (96, 1024, 9000):
        x = torch.randn((50, cols), generator=g, device="cuda")
        gamma = torch.randn(cols, generator=g, device="cuda")
        mean, rstd = torch.empty((2, 50), device="cuda")
        want = torch.empty_like(x)

        def fwd(src, dst, stream=None):
            lc.check(lc.lib.lcLayerNormForward(src.data_ptr(), gamma.data_ptr(), None, dst.data_ptr(), mean.data_ptr(),
                                               rstd.data_ptr(), 50, cols, 0, 0, EPS, lc.F32, lc.F32, stream))

        def bwd(dy, dst, dg, db, stream=None):
            lc.check(lc.lib.lcLayerNormBackward(dy.data_ptr(), x.data_ptr(), gamma.data_ptr(), mean.data_ptr(),
                                                rstd.data_ptr(), dst.data_ptr(), dg.data_ptr(), db.data_ptr(), 50, cols, 0,
                                                0, 0, lc.F32, lc.F32, stream))

        fwd(x, want)
        same = x.clone()
        fwd(same, same)
        torch.cuda.synchronize()
        assert torch.equal(same, want)
        dy = torch.randn((50, cols), generator=g, device="cuda")
        dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
        bwd(dy, dx, dg, db)
        over, dg2, db2 = dy.clone(), torch.empty_like(gamma), torch.empty_like(gamma)
        bwd(over, over, dg2, db2)
        torch.cuda.synchronize()
        assert torch.equal(over, dx) and torch.equal(dg2, dg) and torch.equal(db2, db)
        # Two streams at once, several calls each: every call has its own workspace.
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        outs = [[torch.empty_like(t) for t in (dx, dg, db)] for _ in range(8)]
        torch.cuda.synchronize()
        for i, o in enumerate(outs):
            bwd(dy, *o, stream=streams[i % 2].cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, (dx, dg, db)))
        # Captured once, replayed on new inputs.
        gr = torch.cuda.CUDAGraph()
        y2, o2 = torch.empty_like(x), [torch.zeros_like(t) for t in (dx, dg, db)]
        with torch.cuda.graph(gr):
            s = torch.cuda.current_stream().cuda_stream
            fwd(x, y2, s)
            bwd(dy, *o2, stream=s)
        for _ in range(3):
            for t in o2:
                t.zero_()
            gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(y2, want) and all(torch.equal(a, b) for a, b in zip(o2, (dx, dg, db)))


@pytest.mark.gpu
def test_special_values_stay_in_their_row(gpu):
    """A row with NaN, with an infinity, and a constant row: the others are what they are without them."""
    import torch
    lc = gpu
    x = torch.randn((6, 300), device="cuda")
    want, mean, rstd = lc.layer_norm_affine(x.cpu().numpy())
    y = x.clone()
    y[1, 5], y[2, 0], y[3] = float("nan"), float("inf"), 4.0
    got, m2, r2 = lc.layer_norm_affine(y.cpu().numpy())
    assert np.array_equal(got[[0, 4, 5]], want[[0, 4, 5]])
    assert np.isnan(got[1]).all() and np.isnan(got[2]).any() and not np.any(got[3])
    assert m2[3] == 4.0 and abs(r2[3] * np.sqrt(np.float32(EPS)) - 1) < 4 * U
