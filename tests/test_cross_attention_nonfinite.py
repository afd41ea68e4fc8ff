"""Cross attention where a *visible* query, key, value or gradient is NaN or infinite: what the definition makes NaN
comes out as NaN, what it makes infinite as an infinity (in f32 on the tensor cores as NaN), what it does not
touch keeps its bits, and a masked key's gradient is 0 all the same."""
import pytest

from test_cross_attention import Case

NAN, INF = float("nan"), float("inf")

# name: dtype, layout, (batch, q_heads, kv_heads, q_len, kv_len, head_dim).  One of each kernel, whole and split along
# the keys (batch 1).
FORWARD = {
    "bf16 few 64": ("bf16", "tokens", (2, 4, 2, 1, 200, 64)),
    "bf16 few 128": ("bf16", "tokens", (2, 4, 2, 3, 333, 128)),
    "bf16 few split": ("bf16", "dense", (1, 2, 1, 1, 13000, 64)),
    "bf16 tiled 64": ("bf16", "tokens", (2, 4, 2, 40, 300, 64)),
    "bf16 tiled 72": ("bf16", "tokens", (2, 2, 2, 140, 300, 72)),
    "bf16 tiled 128": ("bf16", "packed", (2, 2, 2, 140, 300, 128)),
    "bf16 tiled split 64": ("bf16", "dense", (1, 1, 1, 17, 3001, 64)),
    "bf16 tiled split 128": ("bf16", "dense", (1, 1, 1, 33, 1500, 128)),
    "bf16 plain": ("bf16", "odd", (2, 4, 2, 20, 150, 40)),
    "bf16 plain split": ("bf16", "dense", (1, 1, 1, 9, 2500, 200)),
    "f32 few 64": ("f32", "tokens", (2, 4, 2, 1, 200, 64)),
    "f32 few 44": ("f32", "tokens", (2, 2, 2, 3, 200, 44)),
    "f32 few 128": ("f32", "tokens", (2, 4, 2, 3, 333, 128)),
    "f32 few split": ("f32", "dense", (1, 2, 1, 1, 13000, 64)),
    "f32 tiled 64": ("f32", "tokens", (2, 4, 2, 40, 300, 64)),
    "f32 tiled 100": ("f32", "odd", (2, 2, 2, 140, 300, 100)),
    "f32 tiled 128": ("f32", "packed", (2, 2, 2, 140, 300, 128)),
    "f32 tiled split 64": ("f32", "dense", (1, 1, 1, 33, 1500, 64)),
    "f32 tiled split 128": ("f32", "dense", (1, 1, 1, 17, 3001, 128)),
    "f32 plain": ("f32", "tokens", (2, 2, 2, 20, 150, 200)),
    "f32 plain few": ("f32", "odd", (2, 2, 2, 3, 150, 64)),
    "f32 plain split": ("f32", "dense", (1, 1, 1, 9, 2500, 200)),
}
BACKWARD = {
    "bf16 tiled 64": ("bf16", "tokens", (2, 4, 2, 140, 300, 64)),
    "bf16 tiled 72": ("bf16", "tokens", (2, 2, 2, 140, 300, 72)),
    "bf16 tiled 128": ("bf16", "packed", (2, 4, 2, 70, 300, 128)),
    "bf16 plain": ("bf16", "odd", (2, 4, 2, 20, 150, 40)),
    "bf16 plain 200": ("bf16", "tokens", (2, 4, 2, 20, 150, 200)),
    "f32 tiled 64": ("f32", "tokens", (2, 4, 2, 140, 300, 64)),
    "f32 tiled 100": ("f32", "odd", (2, 2, 2, 70, 300, 100)),
    "f32 tiled 128": ("f32", "packed", (2, 4, 2, 70, 300, 128)),
    "f32 plain 200": ("f32", "tokens", (2, 4, 2, 20, 150, 200)),
}


def _split_infinities(name):
    """f32 on the tensor cores splits its operands: an infinity is NaN there."""
    return name.startswith("f32 tiled")


def _case(torch, lc, spec, keys="holes", seed=5, **kw):
    """A problem whose masks leave holes; of two batch entries the second sees no key at all."""
    dtype, layout, size = spec
    c = Case(torch, lc, *size, dtype=dtype, layout=layout, seed=seed, **kw)
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = torch.rand((c.b, c.nk), generator=g, device="cuda") < 0.7
    m[:, c.nk // 2] = True
    if c.b > 1:
        m[1] = False
    if keys == "none":
        m[:] = False
    c.key_mask, c.vis = m.to(torch.uint8), m
    hide = ~(m.any(0, keepdim=True) if c.shared else m)
    c.k.masked_fill_(hide[:, None, :, None], NAN)
    c.v.masked_fill_(hide[:, None, :, None], INF)
    return c


def _run(torch, c):
    out, lse = c.forward()
    torch.cuda.synchronize()
    return out.clone(), lse.clone()


def _others(torch, c, hk=0):
    """All rows but those of batch entry 0 that read key head hk, [b, hq, nq]."""
    group = c.hq // c.hk
    other = torch.ones((c.b, c.hq, c.nq), dtype=torch.bool, device="cuda")
    other[0, hk * group:(hk + 1) * group] = False
    return other


def _seen(c):
    """A visible key in the middle."""
    return c.nk // 2


@pytest.mark.gpu
@pytest.mark.parametrize("name", FORWARD)
@pytest.mark.parametrize("value", [NAN, INF])
def test_a_query(gpu, name, value):
    """One value of a row: the row and its log-sum are NaN (inf: +inf and -inf scores), all others keep their bits."""
    import torch
    c = _case(torch, gpu, FORWARD[name])
    want, want_lse = _run(torch, c)
    assert bool(torch.isfinite(want).all()) and bool((want_lse[1:] == -INF).all()) and not bool(want[1:].any())
    h, t = c.hq - 1, c.nq // 2
    c.q[0, h, t, 3] = value
    got, lse = _run(torch, c)
    assert bool(got[0, h, t].isnan().all()) and bool(lse[0, h, t].isnan())
    got[0, h, t], lse[0, h, t] = want[0, h, t], want_lse[0, h, t]
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("name", FORWARD)
def test_rows_without_a_key_stay_zero(gpu, name):
    """NaN in q, and in every key and value: nothing is visible, so the row is 0."""
    import torch
    c = _case(torch, gpu, FORWARD[name], keys="none")
    c.q.fill_(NAN)
    out, lse = _run(torch, c)
    assert not bool(out.any()) and bool((lse == -INF).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", FORWARD)
def test_a_key(gpu, name):
    """A NaN in a visible key: every row that reads its head is NaN, the others keep their bits."""
    import torch
    c = _case(torch, gpu, FORWARD[name])
    want, want_lse = _run(torch, c)
    c.k[0, 0, _seen(c), 5] = NAN
    got, lse = _run(torch, c)
    other = _others(torch, c)
    assert bool(got[~other].isnan().all()) and bool(lse[~other].isnan().all())
    assert torch.equal(got[other], want[other]) and torch.equal(lse[other], want_lse[other])


@pytest.mark.gpu
@pytest.mark.parametrize("name", FORWARD)
def test_a_value(gpu, name):
    """A NaN in a visible value: its column of the rows that read it, and no log-sum."""
    import torch
    c = _case(torch, gpu, FORWARD[name])
    want, want_lse = _run(torch, c)
    c.v[0, 0, _seen(c), 7] = NAN
    got, lse = _run(torch, c)
    other = _others(torch, c)
    assert bool(got[~other][:, 7].isnan().all())
    got[~other] = torch.where(torch.arange(c.d, device="cuda") == 7, want[~other], got[~other])
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("name", FORWARD)
def test_scores_of_minus_infinity(gpu, name):
    """A visible key whose score is -infinity has the weight 0 (in f32 on the tensor cores it is NaN); where all
    visible scores are, there is no softmax: NaN, and not the 0 of a row without a key."""
    import torch
    c = _case(torch, gpu, FORWARD[name])
    c.q[..., 2] = 1.0
    j = _seen(c)
    c.vis[0, j] = False
    c.key_mask[0, j] = 0
    want, want_lse = _run(torch, c)
    c.vis[0, j] = True
    c.key_mask[0, j] = 1
    c.k[0, :, j] = 1.0
    c.k[0, :, j, 2] = -INF
    c.v[0, :, j] = 1.0
    got, lse = _run(torch, c)
    if _split_infinities(name):
        assert bool(got[0].isnan().all()) and bool(lse[0].isnan().all())
    else:
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
    c.k[0, :, :, 2] = torch.where(c.vis[0], -INF, NAN)
    got, lse = _run(torch, c)
    assert bool(got[0].isnan().all()) and bool(lse[0].isnan().all())
    assert not bool(got[1:].any()) and bool((lse[1:] == -INF).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.05, 1.0, 30.0])
@pytest.mark.parametrize("name", ["bf16 few 64", "bf16 tiled 64", "bf16 plain", "f32 few 64", "f32 tiled 64", "f32 plain"])
def test_nan_rows_at_any_scale(gpu, name, scale):
    import torch
    c = _case(torch, gpu, FORWARD[name], scale=scale)
    c.q[0] = NAN
    out, lse = _run(torch, c)
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    assert not bool(out[1:].any()) and bool((lse[1:] == -INF).all())


def _grads(torch, c, out, lse):
    mem, o = c.like(c.dout)
    o.copy_(out)
    g = c.backward(o, lse)
    torch.cuda.synchronize()
    return [x.clone() for x in g]


def _masked_are_zero(torch, c, dk, dv):
    gone = ~c.vis.any(0, keepdim=True) if c.shared else ~c.vis
    gone = gone[:, None, :, None].expand_as(dk)
    assert not bool(dk[gone].ne(0).any()) and not bool(dv[gone].ne(0).any())


@pytest.mark.gpu
@pytest.mark.parametrize("name", BACKWARD)
@pytest.mark.parametrize("value", [NAN, INF])
def test_masked_keys_have_no_gradient(gpu, name, value):
    """Whatever the computed rows of dout, or of q, hold: dk and dv of a masked key are 0."""
    import torch
    c = _case(torch, gpu, BACKWARD[name])
    out, lse = _run(torch, c)
    keep = c.dout.clone()
    c.dout[0, :, c.nq // 3, 6] = value
    dq, dk, dv = _grads(torch, c, out, lse)
    _masked_are_zero(torch, c, dk, dv)
    assert not bool(torch.isfinite(dv[0][:, c.vis[0], 6]).any())
    c.dout.copy_(keep)
    c.q[0, :, c.nq // 2, 1] = value
    out, lse = _run(torch, c)
    dq, dk, dv = _grads(torch, c, out, lse)
    _masked_are_zero(torch, c, dk, dv)


@pytest.mark.gpu
@pytest.mark.parametrize("name", BACKWARD)
def test_rows_without_a_key_have_no_gradient(gpu, name):
    """The batch entry without a visible key: NaN and infinities in its rows of q and dout reach nothing."""
    import torch
    c = _case(torch, gpu, BACKWARD[name])
    out, lse = _run(torch, c)
    want = _grads(torch, c, out, lse)
    c.q[1] = NAN
    c.dout[1] = INF
    c.dout[1, :, 0] = NAN
    again = _run(torch, c)
    got = _grads(torch, c, *again)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    assert not any(bool(g[1].ne(0).any()) for g in got) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("bf16", 36), ("f32", 64), ("f32", 200)])
@pytest.mark.parametrize("value", [NAN, INF])
def test_a_shared_source(gpu, dtype, d, value):
    """One source for the batch: keys that no entry sees have the gradient 0 whatever the rows hold."""
    import torch
    c = _case(torch, gpu, (dtype, "tokens", (3, 4, 2, 30, 200, d)), shared=True)
    out, lse = _run(torch, c)
    c.dout[0, 0, 2, 6] = value
    dq, dk, dv = _grads(torch, c, out, lse)
    _masked_are_zero(torch, c, dk, dv)
    seen = c.vis[0]
    assert not bool(torch.isfinite(dk[0, 0][seen]).any()) and not bool(torch.isfinite(dv[0, 0][seen][:, 6]).any())
    assert not bool(torch.isfinite(dq[0, 0, 2]).any()) and bool(torch.isfinite(dq[1:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", BACKWARD)
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_a_gradient_of_the_output(gpu, name, value):
    """One value of a row of dout: the row of dq, that column of dv and all of dk at the visible keys are not finite;
    masked keys' gradients are 0, and what the row does not reach keeps its bits."""
    import torch
    c = _case(torch, gpu, BACKWARD[name])
    out, lse = _run(torch, c)
    wq, wk, wv = _grads(torch, c, out, lse)
    h, t, col = c.hq - 1, c.nq // 3, 6
    c.dout[0, h, t, col] = value
    dq, dk, dv = _grads(torch, c, out, lse)
    _masked_are_zero(torch, c, dk, dv)
    seen, hk = c.vis[0], c.hk - 1
    assert not bool(torch.isfinite(dq[0, h, t]).any())
    assert not bool(torch.isfinite(dk[0, hk][seen]).any()) and not bool(torch.isfinite(dv[0, hk][seen][:, col]).any())
    dq[0, h, t], dk[0, hk], dv[0, hk, :, col] = wq[0, h, t], wk[0, hk], wv[0, hk, :, col]
    assert torch.equal(dq, wq) and torch.equal(dk, wk) and torch.equal(dv, wv)


@pytest.mark.gpu
@pytest.mark.parametrize("name", BACKWARD)
@pytest.mark.parametrize("value", [NAN, INF])
def test_a_query_and_its_gradients(gpu, name, value):
    """A row of q whose weights are NaN: its dq, and dk and dv of every visible key of its head."""
    import torch
    c = _case(torch, gpu, BACKWARD[name])
    out, lse = _run(torch, c)
    want = _grads(torch, c, out, lse)
    h, t, hk = c.hq - 1, c.nq // 3, c.hk - 1
    c.q[0, h, t, 1] = value
    out, lse = _run(torch, c)
    dq, dk, dv = _grads(torch, c, out, lse)
    _masked_are_zero(torch, c, dk, dv)
    assert bool(dq[0, h, t].isnan().all())
    assert bool(dk[0, hk][c.vis[0]].isnan().all()) and bool(dv[0, hk][c.vis[0]].isnan().all())
    dq[0, h, t], dk[0, hk], dv[0, hk] = want[0][0, h, t], want[1][0, hk], want[2][0, hk]
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", BACKWARD)
def test_a_value_and_its_gradients(gpu, name):
    """A NaN in a visible value: dq of the rows that read it and dk of all that they see; dv does not depend on it."""
    import torch
    c = _case(torch, gpu, BACKWARD[name])
    out, lse = _run(torch, c)
    want = _grads(torch, c, out, lse)
    c.v[0, 0, _seen(c), 4] = NAN
    out, lse = _run(torch, c)
    dq, dk, dv = _grads(torch, c, out, lse)
    _masked_are_zero(torch, c, dk, dv)
    other = _others(torch, c)
    assert bool(dq[~other].isnan().all()) and bool(dk[0, 0][c.vis[0]].isnan().all())
    dk[0, 0] = want[1][0, 0]
    assert torch.equal(dq[other], want[0][other]) and torch.equal(dk, want[1]) and torch.equal(dv, want[2])


@pytest.mark.gpu
@pytest.mark.parametrize("name", FORWARD)
@pytest.mark.parametrize("value", [INF, -INF])
def test_an_infinite_value(gpu, name, value):
    """An infinity in a visible value: every weight is positive, so its column is that infinity (in f32 on the tensor
    cores NaN); a second one of the other sign makes it NaN."""
    import torch
    c = _case(torch, gpu, FORWARD[name], spread=0.5)
    want, want_lse = _run(torch, c)
    c.v[0, 0, _seen(c), 7] = value
    got, lse = _run(torch, c)
    other = _others(torch, c)
    column = got[~other][:, 7]
    assert bool(column.isnan().all() if _split_infinities(name) else (column == value).all())
    got[~other] = torch.where(torch.arange(c.d, device="cuda") == 7, want[~other], got[~other])
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    c.v[0, 0, int(c.vis[0].nonzero()[0]), 7] = -value
    got, _ = _run(torch, c)
    assert bool(got[~other][:, 7].isnan().all())
