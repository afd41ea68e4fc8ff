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
