"""The training-side operators that stand beside the nets, as cases to be measured: layer norm (forward, backward, the weight's
gradient), the global gradient norm with clipping, and an AdamW step over many tensors with its moments in 32 or in 8 bits.

``own = False`` computes them in their plain form (elementary torch operations), ``own = True`` through ``myria3d_amd``.
"""
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LR, BETA1, BETA2, EPS, DECAY, STEPS_DONE, MAX_NORM = 1e-3, 0.9, 0.999, 1e-8, 0.01, 100, 1.0
NORM_EPS = 1e-5
BLOCK = 256  # every tensor's slice of the flat buffers starts at a multiple of this


# ------------------------------------------------------------------------------------------------------------ cases
def _norm(name, rows, cols, dtype, weights="float32", backward=True, pad=0):
    return {"name": name, "op": "layer_norm", "rows": rows, "cols": cols, "dtype": dtype, "weights": weights,
            "backward": backward, "pad": pad}


def _many(name, op, layout, tensors, elements, dtype, bits=32, clip=False):
    case = {"name": name, "op": op, "layout": layout, "tensors": tensors, "elements": elements, "dtype": dtype}
    return {**case, "bits": bits, "clip": clip} if op == "adamw" else case


def listed():
    return [
        # one vector through one norm of a served model: nothing but latency
        _norm("norm_one_row", 1, 1024, "bfloat16", weights="bfloat16", backward=False),
        # an odd width read out of a wider matrix (rows not aligned to anything), trained in fp16
        _norm("norm_ragged", 12801, 515, "float16", pad=3),
        # set-abstraction level 1 of the PointNet++ net in training: 16 tiles x 3 200 centres x 32 neighbours, 64 channels
        _norm("norm_edges", 1638400, 64, "float32"),
        # wide rows in bf16 with fp32 weights: a large hidden state in training
        _norm("norm_wide", 8192, 8192, "bfloat16"),
        # clipping the gradients of the PointNet++ net: 58 tensors, most of them vectors
        _many("clip_pointnet2", "clip", "pointnet2", 58, 0, "float32"),
        # clipping a large net trained in bf16
        _many("clip_large", "clip", "3", 300, 250_000_000, "bfloat16"),
        # the PointNet++ net's optimizer step, moments in 32 bits
        _many("adamw_pointnet2", "adamw", "pointnet2", 58, 0, "float32"),
        # as many tensors as HipRandLANet has, clipped as Lightning's gradient_clip_val would
        _many("adamw_randla", "adamw", "7", 141, 1_112_000, "float32", clip=True),
        # a large net with bf16 parameters, moments in 32 bits, clipped
        _many("adamw_large", "adamw", "11", 300, 150_000_000, "bfloat16", clip=True),
        # the PointNet++ net's optimizer step, moments in 8 bits
        _many("adamw8_pointnet2", "adamw", "pointnet2", 58, 0, "float32", bits=8),
        # a large net whose moments are held in 8 bits to leave the memory to activations, clipped
        _many("adamw8_large", "adamw", "13", 300, 200_000_000, "float32", bits=8, clip=True),
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["layer_norm", "adamw", "adamw", "clip"])
    dtype = rng.choice(list(DTYPES))
    if op == "layer_norm":
        cols = _log(rng, 1, 16384)
        rows = max(1, _log(rng, 1, 100_000_000) // cols)
        case = _norm("", rows, cols, dtype, rng.choice(["float32", dtype]), rng.random() < 0.7, rng.choice([0, 0, 1, 4, 13]))
    else:
        tensors = _log(rng, 1, 400)
        elements = max(tensors, _log(rng, 64, 150_000_000))
        case = _many("", op, str(rng.randrange(1 << 30)), tensors, elements, dtype, rng.choice([32, 8]), rng.random() < 0.5)
    del case["name"]
    return case


def _sizes(case):
    """The tensors' shapes: HipPointNet2(9, 7)'s, or about as many vectors as matrices that share `elements` unevenly."""
    if case["layout"] == "pointnet2":
        mlps = [(12, 32, 32, 64), (67, 64, 64, 128), (131, 128, 128, 256), (384, 128), (192, 64), (73, 64), (64, 64, 32)]
        shapes = []
        for widths in mlps:
            for k, c in zip(widths, widths[1:]):
                shapes += [(c, k), (c,), (c,), (c,)]
        return shapes + [(7, 32), (7,)]
    rng = random.Random(int(case["layout"]))
    left, n = case["elements"], case["tensors"]
    vectors = [min(_log(rng, 1, 4096), max(1, left // n)) for _ in range(n // 2)]
    weights = [rng.random() + 0.05 for _ in range(n - len(vectors))]
    left = max(len(weights), left - sum(vectors))
    shapes = [(v,) for v in vectors]
    for w in weights:
        size = max(1, int(left * w / sum(weights)))
        rows = max(1, int(size ** 0.5) - rng.randrange(3))
        shapes.append((rows, max(1, size // rows)))
    rng.shuffle(shapes)
    return shapes


def _count(shape):
    n = 1
    for s in shape:
        n *= s
    return n


def work(case):
    if case["op"] == "layer_norm":
        e, w = 2 if case["dtype"] != "float32" else 4, 2 if case["weights"] != "float32" else 4
        n = case["rows"] * case["cols"]
        if case["backward"]:  # x and dy in, y and dx out, the weights in, their gradients out
            return {"bytes": 4 * e * n + 4 * w * case["cols"], "flops": 22 * n}
        return {"bytes": 2 * e * n + 2 * w * case["cols"], "flops": 8 * n}
    n, e = sum(_count(s) for s in _sizes(case)), 2 if case["dtype"] != "float32" else 4
    if case["op"] == "clip":
        return {"bytes": 2 * e * n + 4, "flops": 3 * n}
    if case["bits"] == 32:  # p, g, both moments in; p and the moments out
        return {"bytes": (3 * e + 16) * n, "flops": 16 * n}
    # the moments come in as codes with two scales a block, go out as such, and are returned as the values they stand for
    return {"bytes": (3 * e + 4 + 8) * n + 16 * n // BLOCK, "flops": 40 * n}


# ------------------------------------------------------------------------------------------------------------ inputs
def _normal(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "layer_norm":
        rows, cols = case["rows"], case["cols"]
        # activations behind a linear layer: channels with offsets and spreads of their own
        spread = 0.5 + torch.rand(cols, generator=gen, device="cuda")
        wide = torch.zeros((rows, cols + case["pad"]), dtype=dtype, device="cuda")
        wide[:, :cols] = _normal((rows, cols), gen).mul_(spread).add_(0.5 * _normal((cols,), gen)).to(dtype)
        wdtype = DTYPES[case["weights"]]
        state = {"case": case, "x": wide[:, :cols], "w": (1 + 0.2 * _normal((cols,), gen)).to(wdtype),
                 "b": (0.2 * _normal((cols,), gen)).to(wdtype)}
        if case["backward"]:
            state["dy"] = _normal((rows, cols), gen, dtype)
            for k in "xwb":
                state[k].requires_grad_()
        return state
    shapes = _sizes(case)
    starts, at = [], 0
    for s in shapes:
        starts.append(at)
        at += -(-_count(s) // BLOCK) * BLOCK
    # parameters and gradients are views of two buffers, as HipRandLANet.flatten_parameters() lays them out
    flat_p, flat_g = (torch.zeros(at, dtype=dtype, device="cuda") for _ in range(2))
    levels = torch.randn(len(shapes), generator=torch.Generator().manual_seed(seed)).mul_(1.5).exp_().mul_(0.01).tolist()
    params, grads = [], []
    for s, start, level in zip(shapes, starts, levels):
        n = _count(s)
        p, g = (f[start:start + n].view(s) for f in (flat_p, flat_g))
        p.copy_(_normal(s, gen).mul_(0.05))
        v = _normal(s, gen).mul_(level)
        v.mul_(torch.rand(s, generator=gen, device="cuda") > 0.1)  # units that saw nothing in this batch
        g.copy_(v)
        del v
        params.append(p)
        grads.append(g)
    state = {"case": case, "params": params, "flat_p": flat_p, "flat_g": flat_g}
    if case["op"] == "clip":
        state["bound"] = MAX_NORM
    else:  # the moments of a checkpoint that is resumed, in 32 bits
        state["steps"] = STEPS_DONE
        size = flat_g.float().abs_()
        state["m0"] = _normal((at,), gen).mul_(0.3).mul_(size).add_(flat_g.float(), alpha=0.3)
        state["v0"] = torch.rand(at, generator=gen, device="cuda").add_(0.2).mul_(size).mul_(size)
        state["starts"] = starts
    for p, g in zip(params, grads):
        p.requires_grad_()
        p.grad = g
    return state


# ------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if op == "layer_norm":
        return _own_norm(state) if own else _plain_norm(state)
    if op == "clip":
        state["bound"] *= 0.9999  # so that a pass over gradients that are clipped already clips them again
        return _own_clip(state) if own else _plain_clip(state)
    return _own_adamw(state) if own else _plain_adamw(state)


def _own_norm(state):
    from myria3d_amd import layer_norm

    x, w, b = state["x"], state["w"], state["b"]
    y = layer_norm(x, w, b, eps=NORM_EPS)
    if "dy" not in state:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (x, w, b), state["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


@torch.no_grad()
def _plain_norm(state):
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    centred = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + NORM_EPS)
    xh = centred * r
    out = {"y": (xh * w + b).to(state["x"].dtype)}
    if "dy" in state:
        g = state["dy"].float()
        gw = g * w
        gx = g * xh
        dx = r * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
        out |= {"dx": dx.to(state["x"].dtype), "dw": gx.sum(0, dtype=torch.float64).to(state["w"].dtype),
                "db": g.sum(0, dtype=torch.float64).to(state["b"].dtype)}
    return out


def _own_clip(state):
    from myria3d_amd import clip_grad_norm_

    norm = clip_grad_norm_(state["params"], state["bound"])
    return {"norm": norm, "grad": state["flat_g"]}


@torch.no_grad()
def _plain_clip(state):
    g = state["flat_g"]
    norm = g.double().square().sum().sqrt()
    factor = (state["bound"] / (norm + 1e-6)).clamp(max=1.0)
    g.copy_(g.float() * factor.float())
    return {"norm": norm.float(), "grad": g}


def _own_adamw(state):
    from myria3d_amd import AdamW

    case, opt = state["case"], state.get("opt")
    if opt is None:
        opt = state["opt"] = AdamW(state["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                   state_bits=case["bits"], max_grad_norm=MAX_NORM if case["clip"] else None)
        step = torch.tensor(float(state["steps"]))
        moments = [{"step": step, **{k: state[f][a:a + p.numel()].view(p.shape)
                                     for k, f in (("exp_avg", "m0"), ("exp_avg_sq", "v0"))}}
                   for p, a in zip(state["params"], state["starts"])]
        opt.load_state_dict({"state": dict(enumerate(moments)), "param_groups": opt.state_dict()["param_groups"]})
        del state["m0"], state["v0"]
    opt.step()
    (m, v), = opt.moments()
    out = {"param": state["flat_p"], "exp_avg": m, "exp_avg_sq": v}
    return {**out, "norm": opt.grad_norm} if case["clip"] else out


def _nearest_m(m):
    """What a block's first moments are in 8 bits: its largest magnitude, held in 32 bits, times multiples of 2^-8 of what a sign,
    4 bits of exponent and 3 of fraction can say."""
    m = m.view(-1, BLOCK)
    s = m.abs().amax(1, keepdim=True).float()
    s = torch.where(s < 2.0 ** -126, 0, s)
    r = torch.where(s > 0, m / s.double(), 0) * 256
    step = torch.ldexp(torch.ones_like(r), torch.frexp(r)[1].sub_(1).clamp_(min=-6).sub_(3))
    q = (r / step).round().mul_(step)
    return ((q / 256).float() * s).view(-1)


def _nearest_v(v):
    """The same for second moments, in 5 bits of exponent and 3 of fraction: what is above zero stays above it."""
    v = v.view(-1, BLOCK)
    s = v.amax(1, keepdim=True).float()
    s = torch.where(s < 2.0 ** -126, 0, s)
    r = torch.where(s > 0, v / s.double(), 0)
    step = torch.ldexp(torch.ones_like(r), torch.frexp(r)[1].sub_(4))
    q = (r / step).round().mul_(step).clamp_(min=2.0 ** -31 * 1.125)
    return (torch.where(r > 0, q, 0).float() * s).view(-1)


@torch.no_grad()
def _plain_adamw(state):
    case, p, g = state["case"], state["flat_p"], state["flat_g"]
    eight = case["bits"] == 8
    work_type = torch.float64 if eight else torch.float32  # a code may not depend on which side of a border rounding falls
    if "m" not in state:
        m0, v0 = state.pop("m0"), state.pop("v0")
        state["m"], state["v"] = (_nearest_m(m0.double()), _nearest_v(v0.double())) if eight else (m0, v0)
    out = {}
    g = g.to(work_type)
    if case["clip"]:
        norm = g.double().square().sum().sqrt()
        g = g * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).to(work_type)
        out["norm"] = norm.float()
    state["steps"] += 1
    m = state["m"].to(work_type) * BETA1 + g * (1 - BETA1)
    v = state["v"].to(work_type) * BETA2 + g * g * (1 - BETA2)
    size, root = LR / (1 - BETA1 ** state["steps"]), (1 - BETA2 ** state["steps"]) ** 0.5
    p.copy_(p.to(work_type) * (1 - LR * DECAY) - size * m / (v.sqrt() / root + EPS))
    state["m"], state["v"] = (_nearest_m(m), _nearest_v(v)) if eight else (m, v)
    return {"param": p, "exp_avg": state["m"], "exp_avg_sq": state["v"], **out}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"layer_norm": _exact_norm, "clip": _exact_clip, "adamw": _exact_adamw}[case["op"]](case, state)


def _exact_norm(case, state):
    """A slab of rows at a time; the gradient of the row from the Jacobian of x -> (x - mean) / deviation."""
    w, b, n = state["w"].double(), state["b"].double(), case["cols"]
    y = torch.empty((case["rows"], n), dtype=torch.float64, device="cuda")
    dx, dw, db = torch.empty_like(y) if case["backward"] else None, torch.zeros_like(w), torch.zeros_like(b)
    slab = max(1, (1 << 26) // n)
    for a in range(0, case["rows"], slab):
        x = state["x"][a:a + slab].double()
        var, mean = torch.var_mean(x, 1, keepdim=True, unbiased=False)
        deviation = (var + NORM_EPS).sqrt()
        y[a:a + slab] = torch.addcmul(b, (x - mean) / deviation, w)
        if case["backward"]:
            g = state["dy"][a:a + slab].double()
            dw += ((x - mean) / deviation * g).sum(0)
            db += g.sum(0)
            g = g * w
            g = g - g.sum(1, keepdim=True) / n
            along = (g * (x - mean)).sum(1, keepdim=True) / (n * deviation ** 2)
            dx[a:a + slab] = (g - (x - mean) * along) / deviation
    return {"y": y, "dx": dx, "dw": dw, "db": db} if case["backward"] else {"y": y}


def _exact_clip(case, state):
    g = state["flat_g"].double()
    norm = torch.linalg.vector_norm(g)
    bound = state["bound"] * 0.9999
    return {"norm": norm, "grad": g * min(1.0, bound / (float(norm) + 1e-6))}


def _in_table(values, table):
    """Blocks of values as the nearest of `table` (ascending) times the block's largest magnitude, held in 32 bits."""
    blocks = values.view(-1, BLOCK)
    scale = blocks.abs().max(1, keepdim=True).values.float()
    scale[scale < 2.0 ** -126] = 0
    ratio = (blocks / scale.double()).nan_to_num_(0.0, 0.0, 0.0)
    near = table[torch.bucketize(ratio, (table[1:] + table[:-1]) / 2)]
    return near, ratio, scale.double()


def _exact_adamw(case, state):
    g, p, m, v = (state[k].double() for k in ("flat_g", "flat_p", "m0", "v0"))
    eight = case["bits"] == 8
    if eight:
        e4m3 = torch.tensor([f * 2.0 ** -9 for f in range(8)] + [(8 + f) * 2.0 ** (e - 3) for e in range(-6, 9) for f in range(8)],
                            dtype=torch.float64, device="cuda")[:-1] / 256
        signed = torch.cat([-e4m3.flip(0)[:-1], e4m3])
        positive = torch.tensor([0.0] + [2.0 ** ((c >> 3) - 31) * (1 + (c & 7) / 8) for c in range(1, 255)],
                                dtype=torch.float64, device="cuda")

        def held_m(x):
            near, _, scale = _in_table(x, signed)
            return (near * scale).view(-1)

        def held_v(x):
            near, ratio, scale = _in_table(x, positive)
            near = torch.where((ratio > 0) & (near == 0), positive[1], near)
            return (near * scale).view(-1)

        # (what is held is a code times a scale, rounded once more where it is returned: 32 bits)
        m, v = held_m(m).float().double(), held_v(v).float().double()
    out = {}
    if case["clip"]:
        norm = torch.linalg.vector_norm(g)
        out["norm"] = norm
        g = g * min(1.0, MAX_NORM / (float(norm) + 1e-6))
    t = state["steps"] + 1
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g * g - v)
    update = m / (1 - BETA1 ** t) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    p = p - LR * DECAY * p - LR * update
    return {"param": p, "exp_avg": held_m(m) if eight else m, "exp_avg_sq": held_v(v) if eight else v, **out}
