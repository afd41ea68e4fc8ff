"""lcCrossAttentionForward / lcCrossAttentionBackward: calls that are refused."""
import itertools

import pytest

from test_cross_attention import Case, _bwd, _desc, _fwd


@pytest.mark.parametrize("grad,other", itertools.product(("dq", "dk", "dv"), ("dout", "q", "k", "v", "out", "lse")))
def test_refuses_a_gradient_over_an_input(lc, grad, other):
    p = {n: 1024 * (i + 1) for i, n in enumerate(("dout", "q", "k", "v", "out", "lse", "dq", "dk", "dv"))}
    p[grad] = p[other]
    assert _bwd(lc, _desc(lc), **p) == lc.LC_INVALID_VALUE


@pytest.mark.parametrize("one,two", [("dq", "dk"), ("dq", "dv"), ("dk", "dv")])
def test_refuses_one_gradient_over_another(lc, one, two):
    p = {n: 1024 * (i + 1) for i, n in enumerate(("dout", "q", "k", "v", "out", "lse", "dq", "dk", "dv"))}
    p[one] = p[two]
    assert _bwd(lc, _desc(lc), **p) == lc.LC_INVALID_VALUE


@pytest.mark.parametrize("scale", [2.0 ** 127, 3.4e38, -1e-30, float("inf"), float("nan")])
def test_refuses_scales_that_are_no_factor(lc, scale):
    """(Times log2 e they are not finite, and 0 times such a factor is NaN.)"""
    p = {n: 1024 * (i + 1) for i, n in enumerate(("dout", "q", "k", "v", "out", "lse", "dq", "dk", "dv"))}
    assert _fwd(lc, _desc(lc, scale=scale)) == lc.LC_INVALID_VALUE
    assert _bwd(lc, _desc(lc, scale=scale), **p) == lc.LC_INVALID_VALUE


# ---------------------------------------------------------------- GPU
NO_MEMORY = [("bf16", (1, 1, 1, 1, 13000, 64)), ("bf16", (1, 1, 1, 17, 3001, 64)), ("bf16", (1, 1, 1, 9, 2500, 200)),
             ("f32", (1, 1, 1, 1, 13000, 64)), ("f32", (1, 1, 1, 33, 1500, 64)), ("f32", (1, 1, 1, 9, 2500, 200))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", NO_MEMORY)
@pytest.mark.parametrize("after", [0, 1])
def test_forward_without_a_workspace(gpu, dtype, size, after):
    """No room for any workspace (or for the second one): the call takes a slower path that needs none."""
    import torch
    c = Case(torch, gpu, *size, dtype=dtype)
    gpu.lib.lcTestFailAllocations(after, 100)
    try:
        c.forward()
    finally:
        gpu.lib.lcTestFailAllocations(0, 0)
    torch.cuda.synchronize()
    c.check_forward()


@pytest.mark.gpu
@pytest.mark.parametrize("d,shared", [(64, False), (128, False), (200, False), (64, True)])
def test_backward_without_room_for_the_halves(gpu, d, shared):
    """f32: where the split operands do not fit, the CUDA cores take the call; without room for the row terms, an
    error."""
    import torch
    c = Case(torch, gpu, 2, 4, 2, 30, 200, d, keys="lens", layout="tokens", shared=shared)
    out, lse = c.forward()
    torch.cuda.synchronize()
    mem, o = c.like(c.dout)
    o.copy_(out)
    gpu.lib.lcTestFailAllocations(0, 1 if d <= 128 and not shared else 0)
    try:
        grads = c.backward(o, lse)
        torch.cuda.synchronize()
        c.check_backward(o, lse, grads)
        gpu.lib.lcTestFailAllocations(0, 2)
        with pytest.raises(gpu.LightningError):
            c.backward(o, lse)
    finally:
        gpu.lib.lcTestFailAllocations(0, 0)


HOLES = [("bf16", (1, 2, 1, 1, 13000, 64)), ("bf16", (1, 4, 1, 1, 9001, 128)), ("bf16", (1, 1, 1, 17, 3001, 64)),
         ("bf16", (1, 1, 1, 33, 1500, 128)), ("bf16", (1, 1, 1, 9, 2500, 200)), ("bf16", (1, 4, 2, 130, 700, 64)),
         ("bf16", (1, 2, 2, 70, 1000, 128)), ("f32", (1, 2, 1, 1, 13000, 64)), ("f32", (1, 4, 1, 1, 9001, 128)),
         ("f32", (1, 1, 1, 33, 1500, 64)), ("f32", (1, 1, 1, 17, 3001, 128)), ("f32", (1, 1, 1, 9, 2500, 200)),
         ("f32", (1, 4, 2, 130, 700, 64)), ("f32", (1, 2, 2, 70, 1000, 128))]


def _with_mask(torch, c, share, first=0):
    """A mask with a `share` of the keys from `first` on, at random; what it hides holds NaN and infinities."""
    g = torch.Generator(device="cuda").manual_seed(c.nk)
    m = torch.rand((c.b, c.nk), generator=g, device="cuda") < share
    m[:, :first] = False
    m[:, c.nk - 1] = True
    c.key_mask, c.vis = m.to(torch.uint8) * 3, m
    c.k.masked_fill_(~m[:, None, :, None], float("inf"))
    c.v.masked_fill_(~m[:, None, :, None], float("nan"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", HOLES)
@pytest.mark.parametrize("share,first", [(0.6, 0), (0.02, 0), (0.5, 0.8)])
def test_holes_in_the_mask_of_one_entry(gpu, dtype, size, share, first):
    """Scattered visible keys, few of them, and parts of split keys that see none."""
    import torch
    c = Case(torch, gpu, *size, dtype=dtype, layout="tokens")
    _with_mask(torch, c, share, int(first * c.nk))
    out, lse = c.forward()
    torch.cuda.synchronize()
    c.check_forward()
    mem, o = c.like(c.dout)
    o.copy_(out)
    grads = c.backward(o, lse)
    torch.cuda.synchronize()
    c.check_backward(o, lse, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("size", [(2, 4, 2, 70, 300, 64), (2, 2, 1, 130, 257, 128), (2, 2, 2, 20, 90, 200),
                                  (3, 4, 2, 1, 150, 64)])
def test_gradients_of_the_whole_function(gpu, dtype, size):
    """Forward and backward one after the other against 64-bit autograd of the whole function: the backward pass
    reads an `out` that is rounded to the tensors' type and an lse, and both errors enter.

    With u, r, es (scores) and ep (weights) as in test_cross_attention.py: out is off by eo = (p |v|) (4 max es + 2 ep +
    (n + 8) u) + 2 r |out|, lse by el = 2 max es + ep + (n + 4) u + 4 u |lse|.  Hence a weight by a share of rp = 2 es +
    2 ep + 4 u |lse| + el, and ds = p (dP - D) by |ds| (rp + ep) + p ((d + 4) u (|do| |v| + |do| |out|) + |do| eo).  Sums
    over n terms add (n + 8) u of their magnitudes, the result's rounding 2 r of itself."""
    import torch
    c = Case(torch, gpu, *size, dtype=dtype, keys="lens", layout="tokens")
    out, lse = c.forward()
    grads = c.backward(out, lse)
    torch.cuda.synchronize()
    b, hq, hk, nq, nk, d = size
    leaf = lambda x: x.double().nan_to_num(0, 0, 0).requires_grad_()
    q, k, v = leaf(c.q), leaf(c.k), leaf(c.v)
    by = lambda x: x.repeat_interleave(hq // hk, 1)
    hidden = ~c.vis[:, None, None, :]
    s = (q @ by(k).transpose(-1, -2) * c.scale).masked_fill(hidden, -float("inf"))
    p = torch.softmax(s, -1).nan_to_num(0)
    live = c.vis.any(1)[:, None, None, None]
    o = torch.where(live, p, 0) @ by(v)
    want = torch.autograd.grad(o, (q, k, v), c.dout.double(), allow_unused=True)
    want = [w.nan_to_num(0) for w in want]

    U = 2.0 ** -24
    q, k, v, o, p, do = q.detach(), by(k.detach()), by(v.detach()), o.detach(), torch.where(live, p, 0).detach(), c.dout.double()
    _, es = c.scores()
    es = torch.where(hidden, 0, es)
    el2 = torch.logsumexp(s.detach(), -1, keepdim=True).abs().nan_to_num(0, 0, 0)
    n = max(nk, nq * hq // hk)
    top = es.amax(-1, keepdim=True)
    eo = (p @ v.abs()) * (4 * top + 2 * c.ep + (n + 8) * U) + 2 * c.r * o.abs()
    rp = 2 * es + 2 * c.ep + 4 * U * el2 + 2 * top + c.ep + (n + 4) * U + 4 * U * el2
    dp, dd = do @ v.transpose(-1, -2), (do * o).sum(-1, keepdim=True)
    ds = p * (dp - dd)
    eds = ds.abs() * (rp + c.ep) + p * ((d + 4) * U * (do.abs() @ v.abs().transpose(-1, -2) + (do * o).abs().sum(
        -1, keepdim=True)) + (do.abs() * eo).sum(-1, keepdim=True))
    by_key = lambda x: x.reshape(b, hk, hq // hk, nk, d).sum(2)
    more = (n + 8) * U
    tol = [c.scale * (eds @ k.abs() + more * (ds.abs() @ k.abs())),
           by_key(c.scale * (eds.transpose(-1, -2) @ q.abs() + more * (ds.abs().transpose(-1, -2) @ q.abs()))),
           by_key((p * (rp + more)).transpose(-1, -2) @ do.abs())]
    for name, got, w, t in zip(("dq", "dk", "dv"), grads, want, tol):
        off = (got.double() - w).abs() - (t + 2 * c.r * w.abs() + 1e-30)
        assert not bool((off > 0).any()) and bool(torch.isfinite(got).all()), (name, float(off.max()))
