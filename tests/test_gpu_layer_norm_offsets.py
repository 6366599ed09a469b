"""GPU: layer norm of rows far from zero, against its formula in 64 bits.

U = 2^-24 is fp32's half step.  Rounded to a float, the mean of a row is off by up to E = DEPTH U mean|x| (16 elements and one of the rest
a lane, six lane steps, 16 waves), however small the deviations are.  The bounds here are those of a mean that has its rounding error
taken out again: D = |x - mean| in place of |x|, m = mean(D), v the variance.
    x - mu1                  off by U (D + E) at most (exact where x and mu1 are within a factor of two)
    mu2 = mean(x - mu1)      off by (DEPTH + 4) U (m + E): those, its sum, its quotient
    dev = (x - mu1) - mu2    off by U (2 D + E) + (DEPTH + 4) U (m + E) =: e
    sum (x - mu1)^2 - mu2 sum (x - mu1), over cols: for the deviations as they were rounded this is their variance, 2 U (v + m E) from v;
                             the two sums' roundings add (DEPTH + 2) U (v + E^2) and (2 DEPTH + 6) U E (m + E)      =: f
    r                        off by f / (2 (v + eps)) + 4 U of it (scaling, eps, root, quotient)                     =: h
    xh                       off by r e + (h + U) |xh|
Second orders: a hundredth, where the first orders are under one; inputs that break this are not used."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, DEPTH = 2.0 ** -24, 48
# a width for every layout of a row over lanes: 4 to 64 lanes, 128 to 1 024 threads, too wide for registers; some that no vector divides
WIDTHS = [2, 3, 7, 16, 33, 64, 96, 130, 257, 515, 777, 1000, 1024, 2051, 4097, 6000, 8192, 9001, 16384, 17001, 40000]


@pytest.mark.parametrize("dtype, values", [
    (torch.float32, [0.1, 3.3, -1e-3, 3547.8467, -4999.977, 1e6 / 3, 16777215.0, 1e-20 / 3]),
    (torch.bfloat16, [0.1, -3547.8467, 1e6 / 3]), (torch.float16, [0.1, -3547.8467, 65504.0])])
def test_constant_rows_have_no_deviations(dtype, values):
    """The deviations from a mean rounded to a float are a few last places k <= 2 DEPTH + 1 of the constant each; over up to 2^14 columns a
    sum of such whole numbers stays under 2^24 and is exact, and so is its quotient: what is left is 0, y is b and dw is 0.  (Above 2^14
    columns the sum has 53 bits.)"""
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(1)
    for cols in WIDTHS:
        consts = torch.tensor(values, device="cuda").to(dtype)
        x = consts.repeat(5)[:, None].expand(-1, cols).contiguous().requires_grad_()
        w = torch.randn(cols, generator=g, device="cuda", requires_grad=True)
        b = torch.randn(cols, generator=g, device="cuda", requires_grad=True)
        y = myria3d_amd.layer_norm(x, w, b)
        want = b.detach().to(dtype).expand_as(y)
        bad = [float(consts[i % len(values)]) for i in range(len(x)) if not torch.equal(y[i], want[i])]
        assert not bad, (cols, bad)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert not dw.any(), cols
        assert bool((db == len(x)).all()), cols


def bounds(x, w, b, eps, dy):
    """Values of y, dx, dw and db in 64 bits, and what they may be off by."""
    x, w, b, dy = (t.detach().double() for t in (x, w, b, dy))
    mean = x.mean(1, keepdim=True)
    d = x - mean
    E = DEPTH * U * x.abs().mean(1, keepdim=True)
    D, m, v = d.abs(), d.abs().mean(1, keepdim=True), d.square().mean(1, keepdim=True)
    e = U * (2 * D + E) + (DEPTH + 4) * U * (m + E)
    f = U * (2 * (v + m * E) + (DEPTH + 2) * (v + E * E) + (2 * DEPTH + 6) * E * (m + E))
    h = f / (2 * (v + eps)) + 4 * U
    assert float(h.max()) < 0.01 and float((E.square() / v * U).max()) < 1e-4  # (first orders do)
    r = 1 / (v + eps).sqrt()
    xh = d * r
    dxh = 1.01 * (r * e + (h + U) * xh.abs())
    y = xh * w + b
    ey = w.abs() * dxh + 2 * U * (y.abs() + b.abs())
    gw = dy * w
    egw = U * gw.abs()
    m0, m1 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    e0 = (DEPTH + 3) * U * gw.abs().mean(1, keepdim=True)
    e1 = (gw.abs() * dxh).mean(1, keepdim=True) + (DEPTH + 4) * U * (gw * xh).abs().mean(1, keepdim=True)
    dx = r * (gw - m0 - xh * m1)
    edx = 1.01 * (r * (egw + e0 + xh.abs() * e1 + dxh * m1.abs() + 3 * U * (gw.abs() + m0.abs() + (xh * m1).abs())) + (h + 2 * U) * dx.abs())
    rows = x.shape[0]  # (few here: a lane adds up no more than all of them)
    dw, edw = (dy * xh).sum(0), (dy.abs() * dxh + (rows + 8) * U * (dy * xh).abs()).sum(0)
    return {"y": (y, ey), "dx": (dx, edx), "dw": (dw, edw), "db": (dy.sum(0), (rows + 8) * U * dy.abs().sum(0))}


@pytest.mark.parametrize("offset", [0.0, 3e3, -3e4, 1e6])
@pytest.mark.parametrize("cols", [c for c in WIDTHS if c > 3])
def test_an_offset_costs_no_digits(cols, offset):
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(cols)
    x = (torch.randn(70, cols, generator=g, device="cuda") + offset).requires_grad_()
    w = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).requires_grad_()
    b = (0.3 * torch.randn(cols, generator=g, device="cuda")).requires_grad_()
    dy = torch.randn(70, cols, generator=g, device="cuda")
    y = myria3d_amd.layer_norm(x, w, b)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)), y=y.detach())
    for name, (value, bound) in bounds(x, w, b, 1e-5, dy).items():
        worst = ((got[name].double() - value).abs() / bound).max().item()
        assert worst <= 1.0, (name, worst)


def test_both_passes_see_the_same_side_of_the_activation():
    """dy = 1 and slope 0: db counts the rows whose result is above zero, and the forward pass says which these are."""
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(9)
    for cols in (4, 64, 515, 3000, 12000, 17001):
        x = torch.randn(400, cols, generator=g, device="cuda") + 1e5
        w = torch.randn(cols, generator=g, device="cuda")
        b = (-w * 2.0 ** torch.randint(-20, 1, (cols,), generator=g, device="cuda")).requires_grad_()  # (z near zero again and again)
        y = myria3d_amd.layer_norm(x, w, b, negative_slope=0.0)
        (db,) = torch.autograd.grad(y, b, torch.ones_like(y))
        assert torch.equal(db, (y > 0).sum(0).float()), cols


@pytest.mark.parametrize("cols", [1 << 20, 3000001])
def test_sums_over_many_columns(cols):
    """Equal terms add up with roundings of one sign: one thread's thousands of columns in 32 bits would miss the bound three times over."""
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(2)
    x = (torch.randn(3, cols, generator=g, device="cuda") + 100.0).requires_grad_()
    w, b = torch.ones(cols, device="cuda", requires_grad=True), torch.zeros(cols, device="cuda", requires_grad=True)
    dy = torch.full((3, cols), 0.1, device="cuda")
    dy[1] = 0.1 * (x[1].detach() - 100.0) + 0.1
    dy[2] = torch.randn(cols, generator=g, device="cuda")
    y = myria3d_amd.layer_norm(x, w, b)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)), y=y.detach())
    for name, (value, bound) in bounds(x, w, b, 1e-5, dy).items():
        worst = ((got[name].double() - value).abs() / bound).max().item()
        assert worst <= 1.0, (name, worst)
