"""lcLayerNormForward / lcLayerNormBackward written over their inputs: out over x, dx over dout or over x, in rows on and
off the 16-byte grid (whose copies read the neighbouring rows' bytes), several rows to a group.  The same arithmetic
runs in both forms, so the bits are the same."""
import pytest

EPS = 1e-5
# rows x columns: enough rows that every group of an SM's block walks several
SHAPES = [(5000, 64), (5003, 333), (3001, 1333), (1201, 2047), (700, 4099), (400, 8191), (300, 9001), (2048, 1024)]


def _tensors(torch, rows, cols, t, pad, seed):
    """Two tensors with a row stride of cols + pad, and weights."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda: torch.as_strided(torch.randn(rows * (cols + pad), generator=g, device="cuda").to(t), (rows, cols),
                                    (cols + pad, 1))
    return make(), make(), torch.randn(cols, generator=g, device="cuda"), torch.randn(cols, generator=g, device="cuda")


def _copy(torch, x):
    """x with its gaps, in memory of its own."""
    mem = torch.empty(x.shape[0] * x.stride(0), device="cuda", dtype=x.dtype)
    mem.copy_(torch.as_strided(x, mem.shape, (1,), 0))
    return mem, torch.as_strided(mem, x.shape, x.stride(), 0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad", [0, 3])
def test_in_place(gpu, rows, cols, dtype, pad):
    import torch
    lc = gpu
    t, dt = (torch.bfloat16, lc.BF16) if dtype == "bf16" else (torch.float32, lc.F32)
    x, dy, gamma, beta = _tensors(torch, rows, cols, t, pad, rows + cols)
    stride = cols + pad
    mean, rstd = torch.empty((2, rows), device="cuda")

    def forward(src, dst):
        lc.check(lc.lib.lcLayerNormForward(src.data_ptr(), gamma.data_ptr(), beta.data_ptr(), dst.data_ptr(), mean.data_ptr(),
                                           rstd.data_ptr(), rows, cols, stride, stride, EPS, dt, lc.F32, None))

    def backward(dout, src, dx):
        grads = torch.empty((2, cols), device="cuda")
        lc.check(lc.lib.lcLayerNormBackward(dout.data_ptr(), src.data_ptr(), gamma.data_ptr(), mean.data_ptr(),
                                            rstd.data_ptr(), dx.data_ptr(), grads[0].data_ptr(), grads[1].data_ptr(), rows,
                                            cols, stride, stride, stride, dt, lc.F32, None))
        return grads

    want_mem, want = _copy(torch, x)
    torch.cuda.synchronize()
    forward(x, want)
    stats = mean.clone(), rstd.clone()
    same_mem, same = _copy(torch, x)
    torch.cuda.synchronize()
    forward(same, same)
    torch.cuda.synchronize()
    assert torch.equal(same_mem, want_mem) and torch.equal(mean, stats[0]) and torch.equal(rstd, stats[1])

    for over in ("dout", "x"):
        want_mem, dx = _copy(torch, dy if over == "dout" else x)
        torch.cuda.synchronize()
        weights = backward(dy, x, dx)
        torch.cuda.synchronize()
        for _ in range(5):
            mem, same = _copy(torch, dy if over == "dout" else x)
            torch.cuda.synchronize()
            again = backward(same, x, same) if over == "dout" else backward(dy, same, same)
            torch.cuda.synchronize()
            assert torch.equal(mem, want_mem) and torch.equal(again, weights)
