"""GPU: layer norm under tracing and forward-mode differentiation, with and without leaves that require a gradient."""
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu


def _tensors(seed, *shapes):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=g, device="cuda") for s in shapes]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("shape", [(6, 20), (2, 3, 20)])
def test_a_trace_computes(shape, grad):
    import myria3d_amd

    x, z, w, b = _tensors(1, shape, shape, (20,), (20,))
    x.requires_grad_(grad)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # (the checks of the arguments are not part of a trace)
        traced = torch.jit.trace(lambda t: myria3d_amd.layer_norm(t, w, b, negative_slope=0.2) + 1, x, check_trace=False)
    want = myria3d_amd.layer_norm(z, w, b, negative_slope=0.2) + 1
    for _ in range(3):
        torch.full(shape, float("nan"), device="cuda")  # (what an output that nobody writes would find)
        assert torch.equal(traced(z), want)


def test_forward_mode_raises_and_loses_no_tangent():
    import myria3d_amd
    from torch.autograd import forward_ad

    x, t, w, b = _tensors(2, (6, 20), (6, 20), (20,), (20,))
    want = myria3d_amd.layer_norm(x, w, b)
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, t), w, b), (x, forward_ad.make_dual(w, b), b), (x, w, forward_ad.make_dual(b, w))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                myria3d_amd.layer_norm(*args)
        assert torch.equal(myria3d_amd.layer_norm(x, w, b), want)  # no tangent: nothing to lose
    for transform in (lambda f: torch.func.jvp(f, (x,), (t,)), lambda f: torch.func.grad(lambda v: f(v).sum())(x), lambda f: torch.func.vmap(f)(x)):
        with pytest.raises(RuntimeError):
            transform(lambda v: myria3d_amd.layer_norm(v, w, b))
    assert torch.equal(myria3d_amd.layer_norm(x, w, b), want)
