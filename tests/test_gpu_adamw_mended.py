"""GPU: AdamW beside graphs that are still to run, schedulers that go on, groups without parameters and parameters that share memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _param(*shape, seed=0, dtype=torch.float32, grad=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = torch.randn(shape, generator=g, device="cuda").to(dtype).requires_grad_()
    if grad:
        p.grad = torch.randn(shape, generator=g, device="cuda").to(dtype)
    return p


@pytest.mark.parametrize("max_grad_norm", [None, 1.0])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_without_a_gradient_is_not_changed(bits, max_grad_norm):
    """A graph that holds it still runs backward after the step, as with torch's own optimizers."""
    import myria3d_amd

    a, b, c = _param(40, 40, seed=1), _param(40, 40, seed=2, grad=False), _param(300, seed=3)
    opt = myria3d_amd.AdamW([{"params": [a, b]}, {"params": [c]}], lr=1e-2, state_bits=bits, max_grad_norm=max_grad_norm)
    x = torch.randn(8, 40, device="cuda", requires_grad=True)
    pending = (x @ b).square().sum()  # saves b
    was, kept = [p._version for p in (a, b, c)], b.detach().clone()
    wide, far = kept.double(), x.detach().double()
    want, size = 2 * (far @ wide) @ wide.t(), 2 * (far.abs() @ wide.abs()) @ wide.abs().t()
    opt.step()
    assert a._version > was[0] and b._version == was[1] and c._version > was[2]
    pending.backward()
    assert torch.equal(b.detach(), kept)
    assert bool(((x.grad - want).abs() <= 1.01 * (40 + 40 + 1) * U * size).all())  # two products of 40 terms, a doubling
    held = (x @ a).square().sum()
    a.grad, b.grad, c.grad = torch.ones_like(a), None, None
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        held.backward()  # what a step wrote is still noticed
    nothing = [p._version for p in (a, b, c)]
    a.grad = None
    opt.step()
    assert [p._version for p in (a, b, c)] == nothing


@pytest.mark.parametrize("tensor_lr", [False, True])
def test_a_schedule_goes_on_after_loading(tensor_lr):
    """What a scheduler leaves in a group travels with the state, as in torch: here and from torch's own optimizer."""
    import myria3d_amd
    from torch.optim.lr_scheduler import StepLR

    for make in (lambda p: myria3d_amd.AdamW([p], lr=0.5), lambda p: torch.optim.AdamW([p], lr=0.5, betas=(0.8, 0.99))):
        p, q = _param(30, seed=4), _param(30, seed=4)
        first = make(p)
        sched = StepLR(first, 1, 0.5)
        for _ in range(2):
            first.step(), sched.step()
        second = myria3d_amd.AdamW([q], lr=torch.tensor(7.0, device="cuda") if tensor_lr else 7.0)
        second.load_state_dict(first.state_dict())
        assert second.param_groups[0]["betas"] == first.param_groups[0]["betas"]
        again = StepLR(second, 1, 0.5, last_epoch=2)  # (takes its first step by itself)
        sched.step()
        assert again.base_lrs == [0.5] and float(second.param_groups[0]["lr"]) == float(first.param_groups[0]["lr"]) == 0.0625
        saved = second.state_dict()["param_groups"][0]
        assert saved["initial_lr"] == 0.5 and saved["params"] == [0]
    torch.optim.AdamW([q]).load_state_dict(second.state_dict())


def test_weight_decay_stays_of_its_kind():
    """Adam adds its decay to the gradient, AdamW takes it from the parameter: neither goes on as the other without a word."""
    import myria3d_amd

    p, q = _param(30, seed=5), _param(30, seed=5)
    theirs = torch.optim.Adam([p], lr=0.1, weight_decay=0.5)
    theirs.step()
    opt = myria3d_amd.AdamW([q], lr=7.0)
    before = opt.state_dict()
    with pytest.raises(ValueError, match="decay"):
        opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == 7.0 and torch.equal(opt.state_dict()["state"][0]["exp_avg"], before["state"][0]["exp_avg"])
    plain = torch.optim.Adam([p], lr=0.1)  # without decay there is no difference
    plain.step()
    opt.load_state_dict(plain.state_dict())
    assert opt.param_groups[0]["lr"] == 0.1 and opt.param_groups[0]["weight_decay"] == 0.0
    with torch.no_grad():
        q.copy_(p)
    opt.param_groups[0]["weight_decay"] = 0.5
    saved = opt.state_dict()
    other = torch.optim.Adam([p], weight_decay=0.5, foreach=False)
    other.load_state_dict(saved)
    other.step(), opt.step()
    # both decoupled now, each within 16 roundings of p and of an update of at most 10 lr; Adam's own would differ by some 0.1
    assert bool(((p - q).abs() <= 2 * 16 * U * (q.abs() + 1.0)).all())


@pytest.mark.parametrize("bits, max_grad_norm", [(32, None), (8, 0.5)])
def test_groups_without_parameters(bits, max_grad_norm):
    """As torch takes them: in front of, between and behind the others, with a state that travels, and all alone not at all."""
    import myria3d_amd

    p, q = _param(300, seed=6), _param(300, seed=6)
    alone = myria3d_amd.AdamW([q], lr=0.1, state_bits=bits, max_grad_norm=max_grad_norm)
    opt = myria3d_amd.AdamW([{"params": [], "lr": 3.0}, {"params": [p], "lr": 0.1}], state_bits=bits, max_grad_norm=max_grad_norm)
    opt.add_param_group({"params": []})
    for _ in range(2):
        opt.step(), alone.step()
    assert torch.equal(p, q) and [len(g["params"]) for g in opt.param_groups] == [0, 1, 0]
    if max_grad_norm is not None:
        assert torch.equal(opt.grad_norm, alone.grad_norm)
    saved = opt.state_dict()
    assert [g["params"] for g in saved["param_groups"]] == [[], [0], []] and list(saved["state"]) == [0]
    again = myria3d_amd.AdamW([{"params": []}, {"params": [p]}, {"params": []}], state_bits=bits, max_grad_norm=max_grad_norm)
    again.load_state_dict(saved)
    assert [g["lr"] for g in again.param_groups] == [3.0, 0.1, 1e-3]
    again.step(), alone.step()
    assert torch.equal(p, q)
    assert [tuple(m.numel() for m in pair) for pair in again.moments()] == [(0, 0), (512, 512), (0, 0)]
    with pytest.raises(ValueError):
        myria3d_amd.AdamW([{"params": []}, {"params": []}], state_bits=bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_does_not_fit_changes_nothing(bits):
    import copy

    import myria3d_amd

    params = [_param(30, 40, seed=7), _param(700, seed=8)]
    opt = myria3d_amd.AdamW([{"params": params[:1]}, {"params": params[1:]}], lr=0.1, state_bits=bits)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())

    def broken(change):
        d = copy.deepcopy(saved)
        d["param_groups"][0]["lr"] = 0.7
        d["state"][0]["exp_avg"].fill_(3)
        change(d)
        return d

    changes = [lambda d: d["state"][1].pop("exp_avg_sq"), lambda d: d["state"][1].pop("step"),
               lambda d: d["state"][1].update(exp_avg_sq=d["state"][1]["exp_avg_sq"][:1]),  # (one that would spread over all of it)
               lambda d: d["state"][1].update(exp_avg=d["state"][1]["exp_avg"].int()),
               lambda d: d["param_groups"][1].update(betas=(0.9, 1.5)), lambda d: d["param_groups"][1].update(lr=-1.0)]
    if bits == 8:
        changes += [lambda d: d["state"][1].update(exp_avg_scale=d["state"][1]["exp_avg_scale"][:1]),
                    lambda d: d["state"][1].pop("exp_avg_sq_scale"), lambda d: d["state"][1].pop("exp_avg_scale"),
                    lambda d: d["state"][1].update(exp_avg_sq=d["state"][1]["exp_avg_sq"].float())]
    for k, change in enumerate(changes):
        with pytest.raises(ValueError):
            opt.load_state_dict(broken(change))
        now = opt.state_dict()
        assert now["param_groups"] == saved["param_groups"], k
        for i in (0, 1):
            assert all(torch.equal(torch.as_tensor(v), torch.as_tensor(saved["state"][i][name])) for name, v in now["state"][i].items()), (k, i)
    lr = torch.tensor(0.25)  # what torch's capturable optimizers leave in a group
    saved["param_groups"][0].update(lr=lr, betas=[0.5, 0.75])
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["betas"] == (0.5, 0.75)
    opt.step()


def test_parameters_that_share_memory_are_refused():
    """Waves would update the shared elements at the same time, in no order."""
    import myria3d_amd

    flat = torch.zeros(1000, device="cuda")
    a, b, c = (flat[i:j].requires_grad_() for i, j in ((0, 500), (500, 1000), (499, 600)))
    opt = myria3d_amd.AdamW([a, b, torch.zeros(0, device="cuda", requires_grad=True)], lr=0.5)  # neighbours are none
    tied = flat.view(10, 100).requires_grad_()
    for bad in ([a, c], [c, b], [tied, b], [tied, flat[:1000].view(10, 100).requires_grad_()]):
        with pytest.raises(ValueError, match="share"):
            myria3d_amd.AdamW(bad)
        with pytest.raises(ValueError, match="share"):
            opt.add_param_group({"params": [t.detach().requires_grad_() for t in bad]})  # (views of the same memory)
    assert len(opt.param_groups) == 1
    b.data = flat[400:900]
    with pytest.raises(ValueError, match="share"):
        opt.step()
    b.data = flat[500:]
    a.grad, b.grad = torch.ones(500, device="cuda"), -torch.ones(500, device="cuda")
    opt.step()
    assert bool((flat[:500] < -0.4).all()) and bool((flat[500:] > 0.4).all())


def test_what_a_user_keeps_in_a_group_travels_too():
    import myria3d_amd

    p = _param(30, seed=9)
    opt = myria3d_amd.AdamW([{"params": [p], "name": "head", "mask": torch.arange(5.0)}])
    opt.step()
    other = myria3d_amd.AdamW([p])
    saved = opt.state_dict()
    other.load_state_dict(saved)
    group = other.param_groups[0]
    assert group["name"] == "head" and torch.equal(group["mask"], torch.arange(5.0)) and group["mask"] is not saved["param_groups"][0]["mask"]
