"""GPU: the sums over the rows, dw and db, where they are whole numbers: nothing may be lost or counted twice, and no tolerance hides it.

dy is one of -1, 0, 1, 2, the slope 1 or 1 / 2: db is a multiple of 1 / 2, and every partial sum of it is exact in 32 bits up to 2^23.
A row of x holds +a and -a equally often, a a power of two: its mean is 0 exactly, cols a^2 is exact, and over widths with
fl(cols fl(1 / cols)) = 1 the variance is a^2, 1 / deviation (eps = 0) is 1 / a and xh is +1 or -1: dw is such a sum too."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def whole(rows, cols, dtype, slope, seed, pad=0):
    import myria3d_amd

    assert np.float32(cols) * (np.float32(1) / np.float32(cols)) == 1 or cols % 2
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(rows, cols + pad, dtype=dtype, device="cuda")[:, :cols]
    dy = torch.empty(rows, cols + pad, dtype=dtype, device="cuda")[:, :cols]
    at = torch.arange(cols, device="cuda")
    slab = max(1, (1 << 27) // cols)
    for i in range(0, rows, slab):
        n = min(slab, rows - i)
        a = 2.0 ** torch.randint(-3, 4, (n, 1), generator=g, device="cuda")
        turn = torch.randint(0, cols, (n, 1), generator=g, device="cuda")
        x[i:i + n] = torch.where((at + turn) % cols < cols // 2, a, -a).to(dtype)
        dy[i:i + n] = torch.randint(-1, 3, (n, cols), generator=g, device="cuda", dtype=torch.int8).to(dtype)
    x.requires_grad_()
    w = torch.randn(cols, generator=g, device="cuda", requires_grad=True)
    b = torch.randn(cols, generator=g, device="cuda", requires_grad=True)
    y = myria3d_amd.layer_norm(x, w, b, 0.0 if cols % 2 == 0 else 1e-5, slope)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    y = y.detach()
    want_w, want_b = (torch.zeros(cols, dtype=torch.float64, device="cuda") for _ in range(2))
    with torch.no_grad():
        for i in range(0, rows, slab):
            d = dy[i:i + slab].double()
            if slope is not None:
                d = torch.where(y[i:i + slab] > 0, d, d * slope)  # (the side that the forward pass took)
            want_b += d.sum(0)
            want_w += d.mul_(x[i:i + slab].sign()).sum(0)
    assert torch.equal(db, want_b.float()), (db.double() - want_b).abs().max().item()
    if cols % 2 == 0:
        assert torch.equal(dw, want_w.float()), (dw.double() - want_w).abs().max().item()


F32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


# many rows a lane, many partial rows; inside the caches and past them; a whole row in 4 to 64 lanes, in a workgroup, in no registers
@pytest.mark.parametrize("slope", [None, 0.5])
@pytest.mark.parametrize("rows, cols, dtype", [
    (5000001, 6, F32), (7000003, 2, BF16), (3000001, 14, FP16), (6000001, 3, FP16), (1500001, 34, FP16), (1638400, 64, F32), (350001, 100, F32),
    (200003, 130, BF16), (150001, 258, FP16), (100001, 515, F32), (100001, 1024, BF16), (60001, 1500, F32), (40001, 2050, FP16), (20001, 4100, BF16),
    (8000, 8194, F32), (9001, 12000, BF16), (3001, 16384, FP16), (1701, 17000, F32), (1101, 40000, BF16)])
def test_many_rows(rows, cols, dtype, slope):
    whole(rows, cols, dtype, slope, seed=cols)


@pytest.mark.parametrize("cols", [2, 5, 14, 36, 64, 100, 258, 514, 1000, 2050, 5000, 8192, 9000, 12000, 17000])
def test_few_rows(cols):
    for rows in (1, 2, 3, 63, 64, 65, 255, 257, 1025):
        for dtype in (F32, BF16):
            whole(rows, cols, dtype, None, seed=rows)
    whole(999, cols, FP16, 0.5, seed=cols, pad=3)


def test_every_row_beyond_32_bits():
    whole((1 << 31) // 1024 + 1000, 1024, BF16, None, seed=3)


def test_more_columns_than_a_launch_has_threads_for():
    """One column takes 64 threads in the sums over the partial rows: from 2^25 columns on they pass 2^32."""
    whole(3, (1 << 25) + 6, BF16, 0.5, seed=4)
