"""layer_norm_affine / layer_norm_backward of the Python package with bf16 weights."""
import numpy as np
import pytest


def test_refuses_weights_of_another_type(lc):
    x = np.zeros((3, 8), np.float32)
    for bad in (np.ones(8, np.float32), np.ones(7, np.uint16)):
        with pytest.raises(ValueError):
            lc.layer_norm_affine(x, gamma=bad, param_dtype=lc.BF16)
        with pytest.raises(ValueError):
            lc.layer_norm_backward(x, x, np.zeros(3), np.ones(3), gamma=bad, param_dtype=lc.BF16)
    with pytest.raises(ValueError):
        lc.layer_norm_affine(x, gamma=np.ones(8), param_dtype=7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 7, 64, 333])
def test_bf16_weights_are_the_values_they_stand_for(gpu, dtype, cols):
    """The same values in either type give the same bits; the weights' gradients are the fp32 ones rounded once."""
    lc = gpu
    rng = np.random.default_rng(cols)
    x, dy = (rng.standard_normal((5, cols)).astype(np.float32) for _ in range(2))
    gamma, beta = (lc.to_bf16(rng.standard_normal(cols).astype(np.float32)) for _ in range(2))
    wide = lc.from_bf16(gamma), lc.from_bf16(beta)
    dt = lc.F32
    if dtype == "bf16":
        x, dy, dt = lc.to_bf16(x), lc.to_bf16(dy), lc.BF16
    got = lc.layer_norm_affine(x, gamma, beta, dtype=dt, param_dtype=lc.BF16)
    want = lc.layer_norm_affine(x, *wide, dtype=dt)
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    dx, dg, db = lc.layer_norm_backward(dy, x, *got[1:], gamma=gamma, dtype=dt, param_dtype=lc.BF16)
    wx, wg, wb = lc.layer_norm_backward(dy, x, *got[1:], gamma=wide[0], dtype=dt)
    assert np.array_equal(dx, wx) and np.array_equal(dg, lc.to_bf16(wg)) and np.array_equal(db, lc.to_bf16(wb))
