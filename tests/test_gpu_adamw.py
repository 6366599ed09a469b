"""GPU: the global gradient norm, clipping and AdamW over many tensors, against their formulas in 64 bits; a training step of a net
with layer norms that runs them together.

Tolerances count roundings: U = 2^-24 is fp32's half step, a value rounded to a type T is off by half_step(T) of it.  What is held in 8
bits has to be equal: it is defined by operations in 64 bits, one after the other (see M3DAdamW in include/m3d_hip.h)."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

U, BLOCK = 2.0 ** -24, 256
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(1,), (3, 5), (256,), (255,), (257,), (64, 33), (0,), (1000, 7), (2,), (31, 257)]


def half_step(t):
    return torch.finfo(t).eps / 2


def tensors(shapes, dtype, seed, scale=1.0, odd=False):
    """Parameters with gradients; `odd`: views one element behind the start of their storage."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for k, s in enumerate(shapes):
        t = dtype if isinstance(dtype, torch.dtype) else dtype[k % len(dtype)]
        n = 1
        for d in s:
            n *= d
        p, v = (torch.randn(n + odd, generator=g, device="cuda").to(t)[odd:].view(s) for _ in range(2))
        p.requires_grad_()
        p.grad = v * (scale * 10.0 ** (k % 3 - 1))
        if odd:
            buf = torch.empty(n + 1, dtype=t, device="cuda")
            buf[1:] = p.grad.reshape(-1)
            p.grad = buf[1:].view(s)
        out.append(p)
    return out


def grads_of(params):
    return torch.cat([p.grad.detach().double().reshape(-1) for p in params if p.grad is not None])


# ------------------------------------------------------------------------------------------------------------ norm and clipping
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", DTYPES + [DTYPES])
def test_clip_grad_norm(dtype, odd):
    import myria3d_amd

    params = tensors(SIZES * 3, dtype, 1, odd=odd)
    params[4].grad = None
    before = [None if p.grad is None else p.grad.clone() for p in params]
    want = grads_of(params).square().sum().sqrt()
    for bound in (1e9, float(want) / 3, 0.0):
        for p, b in zip(params, before):
            if b is not None:
                p.grad.copy_(b)
        norm = myria3d_amd.clip_grad_norm_(params, bound)
        assert norm.dtype == torch.float32 and norm.shape == ()
        # a 64-bit sum, rounded once
        assert abs(float(norm) - float(want)) <= (U + 1e-12) * float(want)
        k = min(1.0, bound / (float(want) + 1e-6))
        for p, b in zip(params, before):
            if b is None:
                continue
            if k == 1.0:
                assert torch.equal(p.grad, b)
            else:  # the factor and the product in 32 bits, then the type
                exact = b.double() * k
                small = torch.finfo(b.dtype).smallest_normal * half_step(b.dtype) * 2
                assert bool(((p.grad.double() - exact).abs() <= (2.01 * U + half_step(b.dtype) * (b.dtype != torch.float32)) * exact.abs() + small).all())


@pytest.mark.parametrize("shapes", [[(1,)], [(7,)] * 500, [(300, 1000)], [(2000, 3000), (5,), (1,)], [(0,)], [(0,), (3,)] * 200, [(1 << 20,)] * 3])
def test_norm_over_tensor_counts_and_sizes(shapes):
    import myria3d_amd

    for dtype in DTYPES:
        params = tensors(shapes, dtype, 2)
        want = float(grads_of(params).square().sum().sqrt())
        first = [p.grad.clone() for p in params]
        a = myria3d_amd.clip_grad_norm_(params, 0.5)
        got = [p.grad.clone() for p in params]
        for p, f in zip(params, first):
            p.grad.copy_(f)
        b = myria3d_amd.clip_grad_norm_(params, 0.5)
        assert abs(float(a) - want) <= (U + 1e-12) * want
        assert torch.equal(a, b) and all(torch.equal(p.grad, q) for p, q in zip(params, got))  # the same bits every time


def test_norm_of_what_32_bits_cannot_sum():
    """Squares that leave fp32's range, and many small ones beside a large one."""
    import myria3d_amd

    p = torch.zeros(100000, device="cuda", requires_grad=True)
    for big, small in ((1e30, 1.0), (1e-30, 1e-33), (4096.0, 0.25)):
        p.grad = torch.full((100000,), small, device="cuda")
        p.grad[77] = big
        want = p.grad.double().square().sum().sqrt().item()
        assert abs(float(myria3d_amd.clip_grad_norm_(p, 1e38)) - want) <= (U + 1e-12) * want


def test_clip_of_orders_views_and_values_that_are_not_finite():
    import myria3d_amd

    p = torch.zeros(40, 30, device="cuda", requires_grad=True)
    p.grad = torch.randn(30, 40, device="cuda").t()  # dense in another order
    q = torch.zeros(40, 30, device="cuda", requires_grad=True)
    wide = torch.randn(40, 60, device="cuda")
    q.grad = wide[:, ::2]  # not dense: scaled all the same, and only where it is
    keep = wide[:, 1::2].clone()
    a, b = p.grad.clone(), q.grad.clone()
    want = torch.cat([a.reshape(-1), b.reshape(-1)]).double().square().sum().sqrt().item()
    version = q.grad._version
    norm = myria3d_amd.clip_grad_norm_([p, q], want / 2)
    assert abs(float(norm) - want) <= (U + 1e-12) * want and torch.equal(wide[:, 1::2], keep) and q.grad._version > version
    for got, was in ((p.grad, a), (q.grad, b)):
        exact = was.double() * (want / 2 / (want + 1e-6))
        assert bool(((got.double() - exact).abs() <= 2.01 * U * exact.abs() + 1e-40).all())
    r = torch.zeros(300, device="cuda", requires_grad=True)
    r.grad = torch.ones(300, device="cuda")
    r.grad[5] = float("inf")
    assert float(myria3d_amd.clip_grad_norm_(r, 1.0)) == float("inf")
    assert torch.isnan(r.grad[5]) and not r.grad[:5].any() and not r.grad[6:].any()
    r.grad = torch.ones(300, device="cuda")
    r.grad[5] = float("nan")
    assert torch.isnan(myria3d_amd.clip_grad_norm_(r, 1.0)) and bool(torch.isnan(r.grad).all())


def test_clip_beyond_32_bits():
    import myria3d_amd

    n = (1 << 31) + 777
    p = torch.empty(n, dtype=torch.bfloat16, device="cuda").requires_grad_()
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    p.grad[-1000:] = 3.0
    p.grad[:10] = 4.0
    want = (9.0 * 1000 + 160.0) ** 0.5
    norm = myria3d_amd.clip_grad_norm_(p, want / 2)
    assert abs(float(norm) - want) <= 2 * U * want
    assert bool((p.grad[-1000:] == 1.5).all()) and bool((p.grad[:10] == 2.0).all()) and not p.grad[10:2000].any()


# ------------------------------------------------------------------------------------------------------------ AdamW
def table_m():
    e4m3 = [f * 2.0 ** -9 for f in range(8)] + [(8 + f) * 2.0 ** (e - 3) for e in range(-6, 9) for f in range(8)]
    t = torch.tensor(e4m3[:-1], dtype=torch.float64, device="cuda") / 256
    return torch.cat([-t.flip(0)[:-1], t])


def table_v():
    return torch.tensor([0.0] + [2.0 ** ((c >> 3) - 31) * (1 + (c & 7) / 8) for c in range(1, 255)], dtype=torch.float64, device="cuda")


def held(x, table):
    """64-bit values as 8 bits hold them (blocks of 256 from the start of x), decoded in 32 bits."""
    n = x.numel()
    blocks = torch.zeros(-(-max(n, 1) // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    blocks[:n] = x.reshape(-1)
    blocks = blocks.view(-1, BLOCK)
    s = blocks.abs().amax(1, keepdim=True).float()
    s[s < 2.0 ** -126] = 0
    r = torch.where(s > 0, blocks / s.double(), 0.0)
    mids = (table[1:] + table[:-1]) / 2
    at = torch.bucketize(r, mids)  # (a value between two: the lower one)
    zero = int((table == 0).nonzero())
    tie = (r == mids[at.clamp(max=mids.numel() - 1)]) & ((at - zero) % 2 != 0)  # half way (gradients of few bits get there): the even code
    near = table[at + tie]
    if table[0] == 0:  # second moments: what is above zero stays above it
        near = torch.where((r > 0) & (near == 0), table[1], near)
    return (near.float() * s).view(-1)[:n].view(x.shape)


class Oracle:
    """One step in 64 bits from given 32-bit values, with the bounds of what the kernel's 32 bits may differ by."""

    def __init__(self, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        self.lr, self.betas, self.eps, self.wd = lr, betas, eps, weight_decay

    def step(self, p, g, m, v, t, k=1.0):
        b1, b2 = self.betas
        p, g, m, v = p.double(), g.double() * k, m.double(), v.double()
        m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * (g * g)
        # m: two products, a sum, the clipped gradient, the constants: 5 roundings of each term; v: two more, all of one sign
        em, ev = 5 * U * ((b1 * m).abs() + ((1 - b1) * g).abs()), 7 * U * v2
        size, root = self.lr / (1 - b1 ** t), 1 / (1 - b2 ** t) ** 0.5
        denom = v2.sqrt() * root + self.eps
        update = size * m2 / denom
        p2 = p * (1 - self.lr * self.wd) - update
        # the update: m's error, v's halved by the root, and 6 roundings; p: 3 roundings
        ep = size / denom * em + update.abs() * 10 * U + 3 * U * (p.abs() + update.abs())
        return p2, m2, v2, ep, em, ev


def moments_of(opt):
    """(exp_avg, exp_avg_sq) per parameter, in 32 bits, in the parameter's shape."""
    out = []
    for g, (m, v) in zip(opt._groups, opt.moments()):
        out += [(g.slice(m, i).clone(), g.slice(v, i).clone()) for i in range(len(g.params))]
    return out


def check_step(opt, params, oracle, counts, bits, k=1.0):
    """Runs opt.step() and holds every tensor to the oracle's step from the state in front of it."""
    was = [p.detach().clone() for p in params]
    state = moments_of(opt)
    opt.step()
    now = moments_of(opt)
    for i, p in enumerate(params):
        (m0, v0), (m1, v1) = state[i], now[i]
        if p.grad is None:
            assert torch.equal(p, was[i]) and torch.equal(m0, m1) and torch.equal(v0, v1)
            continue
        counts[i] += 1
        p2, m2, v2, ep, em, ev = oracle.step(was[i], p.grad, m0, v0, counts[i], k)
        t = p.dtype
        bound = ep + (half_step(t) * (p2.abs() + ep) if t != torch.float32 else 0.0) + torch.finfo(t).smallest_normal * half_step(t) * 4
        assert bool(((p.detach().double() - p2).abs() <= bound).all()), (i, t)
        if bits == 32:
            assert bool(((m1.double() - m2).abs() <= em + 1e-44).all()) and bool(((v1.double() - v2).abs() <= ev + 1e-44).all()), i
        else:
            assert torch.equal(m1, held(m2, table_m())), i
            assert torch.equal(v1, held(v2, table_v())), i


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", DTYPES + [DTYPES])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_steps(bits, dtype, odd):
    import myria3d_amd

    params = tensors(SIZES, dtype, 3, odd=odd)
    opt = myria3d_amd.AdamW(params, lr=1e-2, state_bits=bits)
    counts = [0] * len(params)
    for step in range(4):
        check_step(opt, params, Oracle(lr=1e-2), counts, bits)
        for p in params:
            p.grad.copy_(torch.randn(p.shape, device="cuda") * 0.1 * (step + 1))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_over_many_tensors_with_clipping(bits):
    """More tensors than a launch holds; a clipped and an unclipped step."""
    import myria3d_amd

    params = tensors([(1 + (37 * k) % 700,) for k in range(400)] + [(0,), (300000,)], DTYPES, 4)
    opt = myria3d_amd.AdamW(params, state_bits=bits, max_grad_norm=1.0)
    counts = [0] * len(params)
    for scale in (1.0, 1e-4):
        for p in params:
            p.grad.mul_(scale)
        grads = [p.grad.clone() for p in params]
        norm = float(grads_of(params).square().sum().sqrt())
        check_step(opt, params, Oracle(), counts, bits, min(1.0, 1.0 / (norm + 1e-6)))
        assert abs(float(opt.grad_norm) - norm) <= (U + 1e-12) * norm
        assert all(torch.equal(p.grad, g) for p, g in zip(params, grads))  # clipped on the way in only
    assert (norm < 1.0) or scale == 1.0


@pytest.mark.parametrize("blocks", [32 * 1290 + 1, 32 * 2100 + 3])  # several chunks of 32 blocks a workgroup; the second: past the caches
@pytest.mark.parametrize("bits, dtype", [(32, torch.float32), (32, torch.bfloat16), (8, torch.float32), (8, torch.float16)])
def test_adamw_over_large_tensors_whose_last_chunk_is_short(bits, dtype, blocks):
    import myria3d_amd

    params = tensors([(BLOCK * 7 - 3,), (BLOCK * (blocks - 9) - 5,), (2 * BLOCK,)], dtype, 14)
    opt = myria3d_amd.AdamW(params, state_bits=bits, max_grad_norm=10.0)
    counts = [0] * 3
    for _ in range(2):
        k = min(1.0, 10.0 / (float(grads_of(params).square().sum().sqrt()) + 1e-6))
        check_step(opt, params, Oracle(), counts, bits, k)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_without_a_gradient_keep_their_own_count(bits):
    import myria3d_amd

    params = tensors([(5,), (300,), (256,), (40, 40)] * 50, torch.float32, 5)
    opt = myria3d_amd.AdamW(params, state_bits=bits)
    counts = [0] * len(params)
    every = [p.grad for p in params]
    for step in range(5):
        for i, p in enumerate(params):
            p.grad = None if (i + step) % 3 == 0 or i == 7 else every[i]
        check_step(opt, params, Oracle(), counts, bits)
    assert [int(s["step"]) for s in opt.state_dict()["state"].values()] == counts and counts[7] == 0


def test_groups_orders_and_a_learning_rate_on_the_device():
    import myria3d_amd

    a, b = tensors([(64, 33), (9,)], torch.float32, 6), tensors([(500,), (31, 257)], torch.bfloat16, 7)
    c = torch.randn(30, 40, device="cuda").t().requires_grad_()  # a dense parameter in another order, its gradient in a third
    c.grad = torch.randn(40, 30, device="cuda")
    lr = torch.tensor(3e-3, device="cuda")
    opt = myria3d_amd.AdamW([{"params": a, "lr": lr}, {"params": b + [c], "weight_decay": 0.0, "betas": (0.5, 0.0), "eps": 1e-3}], lr=1e-2,
                            max_grad_norm=0.1)
    first, second = Oracle(lr=3e-3), Oracle(lr=1e-2, betas=(0.5, 0.0), eps=1e-3, weight_decay=0.0)
    params = a + b + [c]
    for t in (1, 2, 3):
        if t == 3:
            lr.fill_(1e-3)
            first = Oracle(lr=float(lr))
        k = min(1.0, 0.1 / (float(grads_of(params).square().sum().sqrt()) + 1e-6))
        was, state = [p.detach().clone() for p in params], moments_of(opt)
        opt.step()
        for i, p in enumerate(params):
            p2, _, _, ep, _, _ = (first if i < len(a) else second).step(was[i], p.grad, *state[i], t, k)
            bound = ep + half_step(p.dtype) * (p2.abs() + ep)
            assert bool(((p.detach().double() - p2).abs() <= bound).all()), i


def test_codes_say_what_they_stand_for():
    """All values that 8 bits hold, in one block each: taken in and given back unchanged; and halfway cases go to the even code."""
    import myria3d_amd

    tm, tv = table_m(), table_v()
    tm, tv = tm[tm.abs() <= 1.0], tv[tv <= 1.0]
    p = torch.zeros(4 * BLOCK, device="cuda", requires_grad=True)
    opt = myria3d_amd.AdamW([p], state_bits=8)
    for scale in (1.0, 3e-5, 0.7):
        m, v = torch.zeros(4 * BLOCK, device="cuda"), torch.zeros(4 * BLOCK, device="cuda")
        m[:tm.numel()] = tm.float() * torch.tensor(scale)
        m[BLOCK:BLOCK + 1] = scale  # (a block with one value)
        v[:tv.numel()] = tv.float() * torch.tensor(scale)
        entry = {"step": torch.tensor(1.0), "exp_avg": m, "exp_avg_sq": v}
        opt.load_state_dict({"state": {0: entry}, "param_groups": opt.state_dict()["param_groups"]})
        (gm, gv), = opt.moments()
        assert torch.equal(gm, m) and torch.equal(gv, v)
    m, v = torch.zeros(4 * BLOCK, device="cuda"), torch.zeros(4 * BLOCK, device="cuda")
    mid = ((tm[1:] + tm[:-1]) / 2)
    m[:mid.numel()], m[255] = mid.float(), 1.0  # exact in fp32: five significant bits
    midv = ((tv[2:] + tv[1:-1]) / 2)
    v[:midv.numel()], v[255] = midv.float(), 1.0
    v[BLOCK:BLOCK + 3] = torch.tensor([1.0, 2.0 ** -40, 2.0 ** -31], device="cuda")
    entry = {"step": torch.tensor(1.0), "exp_avg": m, "exp_avg_sq": v}
    opt.load_state_dict({"state": {0: entry}, "param_groups": opt.state_dict()["param_groups"]})
    (gm, gv), = opt.moments()
    even = torch.arange(tm.numel(), device="cuda") - tm.numel() // 2  # a code's number: even ones end in an even fraction
    lower = even[:-1].abs() % 2 == 0
    assert torch.equal(gm[:mid.numel()].double(), torch.where(lower, tm[:-1], tm[1:]))
    code = torch.arange(1, tv.numel() - 1, device="cuda")
    assert torch.equal(gv[:midv.numel()].double(), torch.where(code % 2 == 0, tv[1:-1], tv[2:]))
    assert gv[BLOCK + 1].double() == tv[1] and gv[BLOCK + 2].double() == tv[1]  # above zero stays above zero


@pytest.mark.parametrize("bits", [32, 8])
def test_small_values_zeros_and_values_that_are_not_finite(bits):
    import myria3d_amd

    p = torch.ones(6 * BLOCK, device="cuda", requires_grad=True)
    opt = myria3d_amd.AdamW([p], state_bits=bits, weight_decay=0.0)
    p.grad = torch.zeros(6 * BLOCK, device="cuda")
    p.grad[BLOCK:2 * BLOCK] = 1e-37   # moments next to and under the smallest normal number
    p.grad[2 * BLOCK:3 * BLOCK] = 1e-20
    p.grad[3 * BLOCK:] = torch.randn(3 * BLOCK, device="cuda")
    p.grad[3 * BLOCK + 9] = float("inf")
    p.grad[4 * BLOCK + 9] = float("nan")
    good = torch.isfinite(p.grad)
    opt.step()
    assert bool((p[:BLOCK] == 1.0).all()) and bool(torch.isfinite(p[good]).all()) and bool(torch.isnan(p[~good]).all())
    (m, v), = opt.moments()
    assert bool(torch.isfinite(m[good]).all()) and bool(torch.isfinite(v[good]).all())
    assert not bool(torch.isfinite(m[~good]).any()) and not bool(torch.isfinite(v[~good]).any())
    if bits == 8:
        g = torch.where(good, p.grad, 0).double()
        assert torch.equal(m[good], held((1 - 0.9) * g, table_m())[good])
        assert torch.equal(v[good], held((1 - 0.999) * (g * g), table_v())[good])
    if bits == 8:  # (whatever stands beside them, in all places of a word)
        q = torch.ones(300 * BLOCK, device="cuda", requires_grad=True)
        q.grad = torch.randn(300 * BLOCK, device="cuda")
        for k in range(4):
            q.grad[k * BLOCK + k::4 * BLOCK] = (float("inf"), float("nan"), float("-inf"), float("nan"))[k]
        other = myria3d_amd.AdamW([q], state_bits=8)
        other.step()
        (m, v), = other.moments()
        fine = torch.isfinite(q.grad)
        g = torch.where(fine, q.grad, 0).double()
        assert torch.equal(m[fine], held((1 - 0.9) * g, table_m())[fine]) and torch.equal(v[fine], held((1 - 0.999) * (g * g), table_v())[fine])
        assert bool(torch.isnan(m[~fine]).all()) and bool(torch.isnan(v[~fine]).all())
    p.grad.zero_()
    opt.step()  # the others go on
    assert bool(torch.isfinite(p[good]).all()) and bool(torch.isnan(p[~good]).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_whose_norm_is_not_finite_is_not_taken(bits):
    import myria3d_amd

    params = tensors(SIZES * 20, torch.float32, 8)
    opt = myria3d_amd.AdamW(params, state_bits=bits, max_grad_norm=1.0)
    opt.step()
    was, state = [p.detach().clone() for p in params], moments_of(opt)
    skipped = params[3].grad
    for bad in (float("inf"), float("nan")):
        keep = params[5].grad[1, 1].item()
        params[5].grad[1, 1] = bad
        params[3].grad = None
        opt.step()
        assert not torch.isfinite(opt.grad_norm)
        assert all(torch.equal(p, q) for p, q in zip(params, was))
        assert all(torch.equal(a, b) for x, y in zip(moments_of(opt), state) for a, b in zip(x, y))
        assert {int(s["step"]) for s in opt.state_dict()["state"].values()} == {1}
        params[5].grad[1, 1] = keep
        params[3].grad = skipped
    norm = float(grads_of(params).square().sum().sqrt())
    check_step(opt, params, Oracle(), [1] * len(params), bits, min(1.0, 1.0 / (norm + 1e-6)))


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_continues_the_run(bits):
    import myria3d_amd

    params = tensors(SIZES, DTYPES, 9)
    opt = myria3d_amd.AdamW(params, lr=1e-2, state_bits=bits)
    late = params[1].grad
    params[1].grad = None
    opt.step()
    params[1].grad = late
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    if bits == 8:
        assert saved["state"][3]["exp_avg"].dtype == torch.uint8
    twins = [p.detach().clone().requires_grad_() for p in params]
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    other = myria3d_amd.AdamW(twins, lr=5.0, state_bits=bits)
    other.load_state_dict(saved)
    for _ in range(2):
        opt.step(), other.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    assert all(torch.equal(a, b) for x, y in zip(moments_of(opt), moments_of(other)) for a, b in zip(x, y))
    if bits == 8:  # decoded values taken in again give the same codes
        (m, v), = opt.moments()
        g = opt._groups[0]
        plain = {i: {"step": saved["state"][i]["step"], "exp_avg": g.slice(m, i), "exp_avg_sq": g.slice(v, i)} for i in range(len(params))}
        other.load_state_dict({"state": plain, "param_groups": saved["param_groups"]})
        assert torch.equal(other._groups[0].avg, g.avg) and torch.equal(other._groups[0].scale, g.scale)
        assert torch.equal(other._groups[0].avg_sq, g.avg_sq) and torch.equal(other._groups[0].scale_sq, g.scale_sq)
        with pytest.raises(ValueError):
            myria3d_amd.AdamW(twins).load_state_dict(saved)
    with pytest.raises(ValueError):
        myria3d_amd.AdamW(twins[:3], state_bits=bits).load_state_dict(saved)
    with pytest.raises(TypeError):
        copy.deepcopy(opt)
    lr = torch.tensor(0.5, device="cuda")
    there = myria3d_amd.AdamW(twins, lr=lr, state_bits=bits)
    there.load_state_dict(saved)
    assert there.param_groups[0]["lr"] is lr and float(lr) == pytest.approx(1e-2)
    a = torch.zeros(30, 40, device="cuda").requires_grad_()
    b = torch.zeros(40, 30, device="cuda").t().requires_grad_()
    a.grad = torch.randn(30, 40, device="cuda")
    first = myria3d_amd.AdamW([a], state_bits=bits)
    first.step()
    if bits == 8:  # (blocks run along memory)
        with pytest.raises(ValueError):
            myria3d_amd.AdamW([b], state_bits=8).load_state_dict(first.state_dict())
    else:
        second = myria3d_amd.AdamW([b])
        second.load_state_dict(first.state_dict())
        assert torch.equal(moments_of(second)[0][0], moments_of(first)[0][0])


def test_states_travel_to_and_from_torch():
    import myria3d_amd

    params = tensors(SIZES, torch.float32, 10)
    twins = [p.detach().clone().requires_grad_() for p in params]
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    theirs = torch.optim.AdamW(twins, lr=1e-2, foreach=False)
    theirs.step(), theirs.step()
    opt = myria3d_amd.AdamW(params)
    with torch.no_grad():
        for p, q in zip(params, twins):
            p.copy_(q)
    opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == 1e-2
    check_step(opt, params, Oracle(lr=1e-2), [2] * len(params), 32)
    theirs.load_state_dict(opt.state_dict())
    assert all(int(theirs.state[q]["step"]) == 3 for q in twins)
    for q, (m, v) in zip(twins, moments_of(opt)):
        assert torch.equal(theirs.state[q]["exp_avg"], m) and torch.equal(theirs.state[q]["exp_avg_sq"], v)


@pytest.mark.parametrize("bits", [32, 8])
def test_replayed_steps_count_on(bits):
    import myria3d_amd

    params = tensors(SIZES * 18, DTYPES, 11)  # more than one launch
    twins = [p.detach().clone().requires_grad_() for p in params]
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    lr, lr2 = torch.tensor(1e-2, device="cuda"), torch.tensor(1e-2, device="cuda")
    opt = myria3d_amd.AdamW(params, lr=lr, state_bits=bits, max_grad_norm=1.0)
    ref = myria3d_amd.AdamW(twins, lr=lr2, state_bits=bits, max_grad_norm=1.0)
    opt.step(), ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        for p, q in zip(params, twins):
            q.grad.copy_(torch.randn(q.shape, device="cuda"))
            p.grad.copy_(q.grad)
        lr.fill_(1e-2 / (k + 1)), lr2.fill_(1e-2 / (k + 1))
        if k == 2:  # an eager step between two replays
            opt.step()
        else:
            graph.replay()
        ref.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params, twins)), k
        assert torch.equal(opt.grad_norm, ref.grad_norm)
    assert opt.state_dict()["state"][0]["step"] == 5
    side = torch.cuda.Stream()  # another stream than the tensors' own
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    side.synchronize()
    ref.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twins))


def test_clipping_in_a_graph():
    import myria3d_amd

    params = tensors(SIZES * 20, DTYPES, 15)
    myria3d_amd.clip_grad_norm_(params, 1e9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = myria3d_amd.clip_grad_norm_(params, 2.0)
    for k in range(4):
        for p in params:
            p.grad.copy_(torch.randn(p.shape, device="cuda"))
        twins = [p.detach().clone().requires_grad_() for p in params]
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        want = myria3d_amd.clip_grad_norm_(twins, 2.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(p.grad, q.grad) for p, q in zip(params, twins)), k


def test_closures_schedules_scalars_and_groups_that_come_later():
    import myria3d_amd

    a = torch.tensor(2.0, device="cuda", requires_grad=True)  # no dimension
    e = torch.zeros(0, 3, device="cuda", requires_grad=True)  # no element
    opt = myria3d_amd.AdamW([a, e], lr=0.1, weight_decay=0.0)
    late = torch.ones(300, device="cuda", requires_grad=True)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)

    def closure():
        opt.zero_grad()
        loss = a * a + late.sum() + e.sum()
        loss.backward()
        return loss

    assert float(opt.step(closure)) == 304.0
    sched.step()
    assert abs(float(a) - 1.9) <= 16 * U * 2 and not late.ne(1.0).any()  # a first step is lr against the sign
    opt.add_param_group({"params": [late], "lr": 0.25})
    opt.step(closure)
    assert bool(((late - 0.75).abs() <= 16 * U).all())  # its own count: a first step
    assert [int(s["step"]) for s in opt.state_dict()["state"].values()] == [2, 2, 1]
    assert [g["lr"] for g in opt.param_groups] == [0.05, 0.25]
    only = myria3d_amd.AdamW([e], state_bits=8, max_grad_norm=1.0)
    only.step()
    assert float(only.grad_norm) == 0.0 and only.moments()[0][0].numel() == 0
    only.load_state_dict(only.state_dict())
    named = myria3d_amd.AdamW(torch.nn.Linear(3, 2, device="cuda").named_parameters())
    named.step()  # no gradient anywhere: nothing happens
    assert {float(s["step"]) for s in named.state_dict()["state"].values()} == {0.0}


def test_an_eps_under_the_smallest_normal_number_leaves_dead_elements_alone():
    import myria3d_amd

    for bits in (32, 8):
        p = torch.ones(600, device="cuda", requires_grad=True)
        p.grad = torch.zeros(600, device="cuda")
        p.grad[:5] = 1.0
        opt = myria3d_amd.AdamW([p], lr=0.25, eps=1e-42, weight_decay=0.0, state_bits=bits)
        opt.step()
        # the update of a first step is lr against the sign: 14 roundings of a quarter
        assert bool((p[5:] == 1.0).all()) and bool(((p[:5] - 0.75).abs() <= 14 * U).all())


def test_parameters_that_move_and_change():
    import myria3d_amd

    for change, fails in ((lambda p: p.data.clone(), False), (lambda p: p.data.cpu(), True), (lambda p: p.data.double(), True),
                          (lambda p: p.data.t().contiguous().t(), True), (lambda p: p.data.t(), True), (lambda p: torch.zeros(5, 7, device="cuda"), True)):
        p = torch.randn(6, 8, device="cuda", requires_grad=True)
        p.grad = torch.randn(6, 8, device="cuda")
        opt = myria3d_amd.AdamW([p])
        check_step(opt, [p], Oracle(), [0], 32)
        g, p.grad = p.grad, None
        p.data = change(p)
        if fails:
            with pytest.raises((RuntimeError, TypeError)):
                opt.step()
        else:
            p.grad = g
            check_step(opt, [p], Oracle(), [1], 32)


def test_version_counters_and_exchanged_parameters():
    import myria3d_amd

    params = tensors([(4, 4), (7,)], torch.float32, 12)
    opt = myria3d_amd.AdamW(params)
    was = [p._version for p in params]
    opt.step()
    assert all(p._version > v for p, v in zip(params, was))
    opt.param_groups[0]["params"] = params[:1]
    with pytest.raises(RuntimeError):
        opt.step()


def test_adamw_beyond_32_bits():
    import myria3d_amd

    n = (1 << 31) + 1000
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda").requires_grad_()
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    p.grad[-700:] = 2.0
    opt = myria3d_amd.AdamW([p], lr=0.5, state_bits=8, weight_decay=0.0)
    opt.step()
    assert bool((p[-700:] == -0.5).all()) and not p[:-700].any()  # the first step is lr against the gradient's sign


# ------------------------------------------------------------------------------------------------------------ together
def _layer_norm_oracle(num_features, num_classes, k):
    from oracle.pointnet2_oracle import PointNet2Oracle

    ref = PointNet2Oracle(num_features, num_classes, num_neighbors=k, return_logits=True)
    for mlp in [m for m in ref.modules() if hasattr(m, "norms")]:
        for holder in mlp.norms:
            holder.module = torch.nn.LayerNorm(holder.module.num_features)
    return ref


def test_a_training_step_of_a_net_with_layer_norms():
    """HipPointNet2(norm="layer"): logits and every parameter's gradient against the same net in plain torch on the CPU (fp64), then
    clipping and AdamW on them, with moments in 32 and in 8 bits; and its prediction for a tile does not depend on the batch."""
    import myria3d_amd
    from tests._util import fill_params_deterministic, rand_batch

    sizes = [400, 250]
    x, pos, batch, ptr = rand_batch(sizes, seed=3)
    ref = _layer_norm_oracle(9, 6, 8)
    fill_params_deterministic(ref, 2)
    net = myria3d_amd.HipPointNet2(9, 6, num_neighbors=8, return_logits=True, norm="layer")
    net.load_state_dict(ref.state_dict())
    net = net.cuda().train()
    mask = torch.ones(sum(sizes), 32)
    y = torch.randint(0, 6, (sum(sizes),), generator=torch.Generator().manual_seed(1))
    logits = net(x.cuda(), pos.cuda(), batch.cuda(), ptr.cuda(), dropout_mask=mask.cuda())
    loss = myria3d_amd.cross_entropy(logits, y.cuda())
    loss.backward()
    ref32 = copy.deepcopy(ref).train()
    out32 = ref32(x, pos, batch, ptr, dropout_mask=mask)
    torch.nn.functional.cross_entropy(out32, y).backward()
    ref = ref.double().train()
    out = ref(x.double(), pos, batch, ptr, sample_idx=[i.long().cpu() for i in net.last_sample_idx], dropout_mask=mask.double())
    torch.nn.functional.cross_entropy(out, y).backward()
    assert (logits.detach().cpu().double() - out.detach()).abs().max() < 2e-3
    for (name, p), q, q32 in zip(net.named_parameters(), ref.parameters(), ref32.parameters()):
        # a max over neighbours may choose another of two that are equal to 32 bits: the same net in 32 bits on the CPU shows by how
        # much that moves a gradient, beside the 2e-3 that holds for this net's gradients with batch norm
        scale = q.grad.norm().item() + 1e-6
        own = (q32.grad.double() - q.grad).norm().item() / scale
        assert (p.grad.cpu().double() - q.grad).norm().item() / scale <= 2e-3 + 2 * own, name
    for bits in (32, 8):
        twin = copy.deepcopy(net)
        for p, q in zip(twin.parameters(), net.parameters()):
            p.grad = q.grad.clone()
        opt = myria3d_amd.AdamW(twin.parameters(), lr=1e-3, state_bits=bits, max_grad_norm=0.5)
        params = list(twin.parameters())
        norm = float(grads_of(params).square().sum().sqrt())
        check_step(opt, params, Oracle(), [0] * len(params), bits, min(1.0, 0.5 / (norm + 1e-6)))
        assert float(opt.grad_norm) == pytest.approx(norm, rel=1e-6)
        assert float(myria3d_amd.clip_grad_norm_(params, 0.5)) == float(opt.grad_norm)
        opt.zero_grad()
        myria3d_amd.cross_entropy(twin(x.cuda(), pos.cuda(), batch.cuda(), ptr.cuda()), y.cuda()).backward()
        opt.step()
        assert all(bool(torch.isfinite(p).all()) for p in params)
    net.eval()
    with torch.no_grad():
        both = net(x.cuda(), pos.cuda(), batch.cuda(), ptr.cuda())
        one = net(x[:400].cuda(), pos[:400].cuda(), batch[:400].cuda(), ptr[:2].cuda())
    assert (both[:400] - one).abs().max().item() < 1e-5
    net.matmul_precision = "bf16"
    with pytest.raises(ValueError):
        net(x.cuda(), pos.cuda(), batch.cuda(), ptr.cuda())


def test_clipping_serves_the_flat_optimizer_too():
    """clip_grad_norm_ between backward() and FusedAdam.step(): the flat gradients are scaled in place."""
    import myria3d_amd
    from tests._util import rand_batch

    x, pos, batch, ptr = (t.cuda() for t in rand_batch([500, 300], seed=5))
    net = myria3d_amd.HipRandLANet(9, 6, return_logits=True).cuda().train().flatten_parameters()
    opt = myria3d_amd.FusedAdam(net, lr=1e-3)
    y = torch.randint(0, 6, (800,), device="cuda")
    myria3d_amd.cross_entropy(net(x, pos, batch, ptr), y).backward()
    opt.reduce_gradients()
    flat = net.flat_grads.clone()
    want = flat.double().square().sum().sqrt().item()
    norm = myria3d_amd.clip_grad_norm_(net.parameters(), want / 4)
    assert abs(float(norm) - want) <= 2 * U * want
    exact = flat.double() * (want / 4 / (want + 1e-6))
    assert bool(((net.flat_grads.double() - exact).abs() <= 2.01 * U * exact.abs() + 1e-40).all())
    opt.step()
