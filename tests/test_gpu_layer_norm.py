"""GPU: layer norm, forward and backward, against its formula in 64 bits.

Tolerances are the roundings' own.  U = 2^-24 is fp32's half step; a sum of a row is at most DEPTH additions deep (16 elements and
one of the rest a lane, six lane steps, 16 waves; the widest rows: 20 elements a thread), so
    |mean' - mean|  <= DEPTH U mean|x|            xh = (x - mean) r  is then off by  r DEPTH U mean|x| + (DEPTH + 8) U |xh|
(the variance: 2 roundings an element, the sum, the shifted mean in second order; r: half of that and a root and a quotient).
y adds two roundings of its size and the half step of its type; the gradients' bounds follow the same way, term by term."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, DEPTH = 2.0 ** -24, 48
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def reference(x, w, b, eps, slope, dy=None):
    """Values in 64 bits and the bounds of their errors."""
    x = x.double()
    w = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    r = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * r
    dxh = r * DEPTH * U * x.abs().mean(1, keepdim=True) + (DEPTH + 8) * U * xh.abs() + (r * DEPTH * U * x.abs().mean(1, keepdim=True)) ** 2 * xh.abs()
    z = xh * w + b
    dz = w.abs() * dxh + 2 * U * (z.abs() + b.abs())
    y = torch.where(z > 0, z, z * slope)
    out = {"y": (y, dz * max(1.0, slope) + U * y.abs())}
    if dy is None:
        return out
    g = dy.double()
    border = z.abs() <= dz if slope != 1.0 else torch.zeros_like(z, dtype=torch.bool)  # (either side of the activation is right)
    dg = torch.where(border, g.abs() * abs(1 - slope), U * g.abs())
    g = torch.where(z > 0, g, g * slope)
    gw = g * w
    dgw = dg * w.abs() + U * gw.abs()
    m0, m1 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    e0 = dgw.mean(1, keepdim=True) + (DEPTH + 2) * U * gw.abs().mean(1, keepdim=True)
    e1 = (dgw * xh.abs() + gw.abs() * dxh).mean(1, keepdim=True) + (DEPTH + 3) * U * (gw * xh).abs().mean(1, keepdim=True)
    inner = gw - m0 - xh * m1
    dr = (DEPTH + 8) * U + (r * DEPTH * U * x.abs().mean(1, keepdim=True)) ** 2
    dx = r * inner
    edx = r * (dgw + e0 + xh.abs() * e1 + dxh * m1.abs() + 3 * U * (gw.abs() + m0.abs() + (xh * m1).abs())) + dr * dx.abs() + U * dx.abs()
    rows = x.shape[0]
    out["dx"] = dx, edx
    out["dw"] = (g * xh).sum(0), (dg * xh.abs() + g.abs() * dxh + (rows + 8) * U * (g * xh).abs()).sum(0)
    out["db"] = g.sum(0), (dg + (rows + 8) * U * g.abs()).sum(0)
    return out


def check(got, name, ref, dtype):
    value, bound = ref[name]
    bound = bound + half_step(dtype) * (value.abs() + bound) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 4
    got = got.double()
    assert got.shape == value.shape
    assert bool(torch.isfinite(got).all()), name
    worst = ((got - value).abs() / bound.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, (name, worst)


def run_case(rows, cols, dtype, wtype, slope=None, offset=0.0, seed=0, pad=0, weight=True, bias=True):
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = (torch.randn(rows, cols + pad, generator=g, device="cuda") + offset).to(dtype)
    x = wide[:, pad // 2:pad // 2 + cols].requires_grad_()
    w = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(wtype).requires_grad_() if weight else None
    b = (0.3 * torch.randn(cols, generator=g, device="cuda")).to(wtype).requires_grad_() if bias else None
    dy = torch.randn(rows, cols, generator=g, device="cuda").to(dtype)
    y = myria3d_amd.layer_norm(x, w, b, 1e-5, slope)
    with torch.no_grad():
        assert torch.equal(y, myria3d_amd.layer_norm(x, w, b, 1e-5, slope))  # without statistics: the same bits
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # a fixed order of all sums
    with torch.no_grad():
        ref = reference(x, w, b, 1e-5, 1.0 if slope is None else slope, dy)
    check(y.detach(), "y", ref, dtype)
    names = ["dx"] + (["dw"] if weight else []) + (["db"] if bias else [])
    for name, got, leaf in zip(names, grads, leaves):
        assert got.dtype == leaf.dtype
        check(got, name, ref, leaf.dtype)


# every layout of a row over lanes (8 to 64 lanes, 128 to 1 024 threads, too wide for registers), on, under and over its border, and
# widths that no vector divides
@pytest.mark.parametrize("cols", [1, 3, 4, 7, 8, 9, 31, 32, 64, 127, 128, 129, 255, 257, 512, 515, 1000, 1024, 1025, 2048, 2051, 4097, 8192, 8193,
                                  16384, 16387, 20011])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_width(cols, dtype):
    run_case(37 if cols > 600 else 301, cols, dtype, torch.float32, seed=cols)


@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 64), (1, 4096), (2, 130), (7, 8), (33, 64), (5000, 64), (4099, 32), (3000, 300), (1500, 2049)])
@pytest.mark.parametrize("dtype, wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                          (torch.float16, torch.float32), (torch.float32, torch.bfloat16)])
def test_row_counts_and_weight_types(rows, cols, dtype, wtype):
    run_case(rows, cols, dtype, wtype, seed=rows)


@pytest.mark.parametrize("rows, cols, dtype", [(350001, 100, torch.float32), (20001, 4100, torch.bfloat16), (1500001, 33, torch.float16),
                                               (8000, 9000, torch.float32)])
def test_what_the_caches_do_not_hold(rows, cols, dtype):
    run_case(rows, cols, dtype, torch.float32, slope=0.2, seed=rows)


@pytest.mark.parametrize("pad", [1, 2, 5, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_with_a_stride_of_their_own(pad, dtype):
    for cols in (5, 64, 515, 3000):
        run_case(65, cols, dtype, torch.float32, pad=pad, seed=cols + pad)


@pytest.mark.parametrize("cols", [6, 64, 300, 1500, 5000, 12000, 17000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_with_the_activation_behind_it(cols, dtype):
    run_case(130, cols, dtype, torch.float32, slope=0.2, seed=cols)
    run_case(130, cols, dtype, torch.float32, slope=0.0, seed=cols + 1)


@pytest.mark.parametrize("offset", [100.0, -3e3])
def test_a_common_offset_costs_no_digits_beyond_the_means_own(offset):
    for cols in (12, 64, 700, 5000):
        run_case(64, cols, torch.float32, torch.float32, offset=offset, seed=cols)


@pytest.mark.parametrize("weight, bias", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(weight, bias):
    for cols in (5, 64, 2100):
        run_case(50, cols, torch.float32, torch.float32, weight=weight, bias=bias, seed=cols)
        run_case(50, cols, torch.bfloat16, torch.float32, weight=weight, bias=bias, slope=0.2, seed=cols)


def test_shapes_orders_and_empty_batches():
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(1)
    w, b = (torch.randn(12, generator=g, device="cuda", requires_grad=True) for _ in range(2))
    base = torch.randn(5, 12, 7, generator=g, device="cuda")
    x = base.transpose(1, 2).requires_grad_()  # the normalised dimension is not the innermost one
    y = myria3d_amd.layer_norm(x, w, b)
    assert y.shape == (5, 7, 12)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones((), device="cuda").expand(5, 7, 12))  # (the gradient of a sum)
    with torch.no_grad():
        ref = reference(x.reshape(-1, 12), w, b, 1e-5, 1.0, torch.ones(35, 12, device="cuda"))
    check(y.detach().reshape(-1, 12), "y", ref, torch.float32)
    check(dx.reshape(-1, 12), "dx", ref, torch.float32)
    check(dw, "dw", ref, torch.float32), check(db, "db", ref, torch.float32)
    row = torch.randn(1, 12, generator=g, device="cuda", requires_grad=True)  # a broadcast row: its gradient sums over the copies
    dy = torch.randn(9, 12, generator=g, device="cuda")
    (drow,) = torch.autograd.grad(myria3d_amd.layer_norm(row.expand(9, 12), w, b), row, dy)
    with torch.no_grad():
        value, bound = reference(row.expand(9, 12), w, b, 1e-5, 1.0, dy)["dx"]
    assert bool(((drow.double() - value.sum(0)).abs() <= bound.sum(0) + 16 * U * value.abs().sum(0)).all())
    for shape in ((0, 12), (3, 0, 12)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        y = myria3d_amd.layer_norm(e, w, b)
        assert y.shape == shape
        dx, dw, db = torch.autograd.grad(y.sum(), (e, w, b))
        assert dx.shape == shape and not dw.any() and not db.any()
    v = torch.randn(12, generator=g, device="cuda")  # a single vector
    assert torch.equal(myria3d_amd.layer_norm(v, w, b), myria3d_amd.layer_norm(v[None], w, b)[0])


def test_rows_that_are_constant_and_rows_that_are_not_finite():
    import myria3d_amd

    for cols in (1, 5, 64, 777, 5000, 17001):
        x = torch.randn(70, cols, device="cuda")
        x[3] = 7.25  # variance 0: xh = 0 exactly (its mean is exact), y = b, dx = r (g w - mean(g w))
        x[11, cols // 2] = float("inf")
        x[12, 0] = float("nan")
        w, b = torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
        y = myria3d_amd.layer_norm(x, w, b)
        assert torch.equal(y[3], b)
        bad = torch.zeros(70, dtype=torch.bool, device="cuda")
        bad[11] = bad[12] = True
        assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[~bad]).all())
        xg = x.clone().requires_grad_()
        wg, bg = w.clone().requires_grad_(), b.clone().requires_grad_()
        dy = torch.randn(70, cols, device="cuda")
        dx, dw, db = torch.autograd.grad(myria3d_amd.layer_norm(xg, wg, bg), (xg, wg, bg), dy)
        assert bool(torch.isfinite(dx[~bad]).all()) and bool(torch.isnan(dx[bad]).all()) and bool(torch.isfinite(db).all())


def test_gradients_against_differences():
    """The formula's own gradient, by central differences in 64 bits on the formula, and the kernel's against it."""
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(3, 10, generator=g, device="cuda", requires_grad=True)
    w = torch.randn(10, generator=g, device="cuda", requires_grad=True)
    b = torch.randn(10, generator=g, device="cuda", requires_grad=True)
    dy = torch.randn(3, 10, generator=g, device="cuda")
    grads = torch.autograd.grad(myria3d_amd.layer_norm(x, w, b, 1e-3), (x, w, b), dy)

    def loss(x, w, b):
        d = x - x.mean(1, keepdim=True)
        return (dy.double() * (d / (d.square().mean(1, keepdim=True) + 1e-3).sqrt() * w + b)).sum().item()

    at = [t.detach().double() for t in (x, w, b)]
    h = 1e-5
    for k, got in enumerate(grads):
        for i in range(0, got.numel(), 3):
            lo, hi = [t.clone() for t in at], [t.clone() for t in at]
            lo[k].view(-1)[i] -= h
            hi[k].view(-1)[i] += h
            d = (loss(*hi) - loss(*lo)) / (2 * h)
            # differences: h^2 times a third derivative of order 100, 1e-8, and 2^-53 / h, 1e-10; the kernel: some 100 U of terms of order 10
            assert abs(got.view(-1)[i].item() - d) <= 1e-8 + 1e-10 + 1000 * U, (k, i)


def test_only_the_gradients_that_are_asked_for():
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(4)
    for cols in (64, 5000):
        x, w, b = (torch.randn(s, generator=g, device="cuda", requires_grad=True) for s in ((40, cols), (cols,), (cols,)))
        dy = torch.randn(40, cols, generator=g, device="cuda")
        every = torch.autograd.grad(myria3d_amd.layer_norm(x, w, b, negative_slope=0.2), (x, w, b), dy)
        for k, leaf in enumerate((x, w, b)):
            args = [t if t is leaf else t.detach() for t in (x, w, b)]
            (one,) = torch.autograd.grad(myria3d_amd.layer_norm(*args, negative_slope=0.2), leaf, dy)
            assert torch.equal(one, every[k])


def test_a_second_derivative_is_refused_and_inference_runs():
    import myria3d_amd

    x, w = torch.randn(4, 16, device="cuda", requires_grad=True), torch.randn(16, device="cuda", requires_grad=True)
    y = myria3d_amd.layer_norm(x, w)
    (plain,) = torch.autograd.grad(y.square().sum(), x, retain_graph=True)
    (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    assert torch.equal(dx, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)
    with torch.inference_mode():
        assert torch.equal(myria3d_amd.layer_norm(x, w), y.detach())


def test_offsets_beyond_32_bits():
    import myria3d_amd

    cols = 1024
    rows = (1 << 31) // cols + 1000  # over 2^31 elements, 2^32 bytes
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-2000:] = torch.randn(2000, cols, device="cuda").to(torch.bfloat16)
    x[:-2000] = 1.0
    x.requires_grad_()
    w = torch.randn(cols, device="cuda", requires_grad=True)
    b = torch.randn(cols, device="cuda", requires_grad=True)
    y = myria3d_amd.layer_norm(x, w, b)
    dy = torch.zeros_like(y)
    dy[-2000:] = torch.randn(2000, cols, device="cuda").to(torch.bfloat16)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        ref = reference(x[-2000:], w, b, 1e-5, 1.0, dy[-2000:])
    check(y[-2000:].detach(), "y", ref, torch.bfloat16)
    check(dx[-2000:], "dx", ref, torch.bfloat16)
    check(dw, "dw", ref, torch.float32), check(db, "db", ref, torch.float32)


def test_on_another_stream_and_in_a_graph():
    import myria3d_amd

    g = torch.Generator(device="cuda").manual_seed(5)
    x, w, b = (torch.randn(s, generator=g, device="cuda", requires_grad=True) for s in ((700, 96), (96,), (96,)))
    dy = torch.randn(700, 96, generator=g, device="cuda")

    def step():
        y = myria3d_amd.layer_norm(x, w, b, negative_slope=0.2)
        return (y, *torch.autograd.grad(y, (x, w, b), dy))

    def fresh(seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            for t in (x, w, b, dy):
                t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.detach() for t in step()]
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [t.detach() for t in step()]
    for seed in range(4):  # replays on new values in the same place, with eager work between them
        fresh(seed)
        want = [t.detach().clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want)), seed
