"""lcCrossAttentionForward / lcCrossAttentionBackward: calls that are refused."""
import itertools

import pytest

from test_cross_attention import _bwd, _desc, _fwd


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
