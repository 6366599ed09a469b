"""CPU: what the training-side operators (layer norm, gradient clipping, AdamW over many tensors) refuse, and their entry points'
error codes — none of these calls reaches a launch."""
import ctypes
from array import array

import pytest
import torch

import myria3d_amd
from myria3d_amd import _lib

P = 4096  # a well-aligned address that no refused call reads


def test_layer_norm_refuses_what_it_does_not_compute():
    x, w = torch.zeros(4, 8), torch.ones(8)
    for bad, err in (((x.double(), w, w), TypeError), ((x, w.double(), None), TypeError), ((x, torch.ones(7), None), ValueError),
                     ((x, None, torch.ones(8, 1)), ValueError), ((x, torch.ones(16)[::2], None), ValueError),
                     ((x, w, w.to(torch.bfloat16)), TypeError), ((torch.zeros(4, 0), None, None), ValueError),
                     ((torch.zeros(()), None, None), ValueError), ((x.int(), None, None), TypeError)):
        with pytest.raises(err):
            myria3d_amd.layer_norm(*bad)
    with pytest.raises(ValueError):
        myria3d_amd.layer_norm(x, w, w, eps=-1.0)
    with pytest.raises(ValueError):
        myria3d_amd.layer_norm(x, w, w, eps=float("nan"))
    for slope in (-0.1, float("nan")):
        with pytest.raises(ValueError):
            myria3d_amd.layer_norm(x, w, w, negative_slope=slope)
    with pytest.raises(RuntimeError, match="MI355X"):
        myria3d_amd.layer_norm(x, w, w)


def _with_grad(*shape, dtype=torch.float32):
    p = torch.zeros(shape, dtype=dtype, requires_grad=True)
    p.grad = torch.ones_like(p)
    return p


def test_clip_grad_norm_refuses():
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            myria3d_amd.clip_grad_norm_([_with_grad(3)], bad)
    with pytest.raises(TypeError):
        myria3d_amd.clip_grad_norm_([_with_grad(3, dtype=torch.float64)], 1.0)
    p = _with_grad(3)
    with pytest.raises(ValueError):
        myria3d_amd.clip_grad_norm_([p, p], 1.0)
    s = torch.zeros(4, 2, requires_grad=True)
    s.grad = torch.zeros(4, 2).to_sparse()
    with pytest.raises(RuntimeError):
        myria3d_amd.clip_grad_norm_([s], 1.0)
    with pytest.raises(RuntimeError, match="MI355X"):
        myria3d_amd.clip_grad_norm_([_with_grad(3)], 1.0)
    assert float(myria3d_amd.clip_grad_norm_([torch.zeros(3, requires_grad=True)], 1.0)) == 0.0  # no gradient: nothing to scale
    assert float(myria3d_amd.clip_grad_norm_([], 1.0)) == 0.0


@pytest.mark.parametrize("kw, err", [
    ({"state_bits": 16}, ValueError), ({"max_grad_norm": -1.0}, ValueError), ({"lr": -1.0}, ValueError), ({"lr": float("inf")}, ValueError),
    ({"betas": (1.0, 0.999)}, ValueError), ({"betas": (0.9, -0.1)}, ValueError), ({"eps": -1e-8}, ValueError),
    ({"weight_decay": -0.1}, ValueError), ({"state_bits": 8, "eps": 0.0}, ValueError), ({"lr": torch.zeros(())}, ValueError), ({}, RuntimeError)])
def test_adamw_refuses_hyperparameters(kw, err):
    with pytest.raises(err):
        myria3d_amd.AdamW([torch.zeros(4, requires_grad=True)], **kw)


def test_adamw_refuses_parameters():
    p = torch.zeros(4, 6, requires_grad=True)
    for bad, err in (([torch.zeros(4, dtype=torch.float64, requires_grad=True)], TypeError),
                     ([torch.zeros(4, 6)[:, ::2].requires_grad_()], ValueError), ([{"params": [p, p]}], ValueError),
                     ([{"params": []}], ValueError), ([p], RuntimeError)):
        with pytest.raises(err):
            myria3d_amd.AdamW(bad)


def test_dense_orders():
    from myria3d_amd.train import _dense

    t = torch.zeros(3, 4, 5)
    assert _dense(t) and _dense(t.transpose(0, 2)) and _dense(t.permute(1, 2, 0)) and _dense(torch.zeros(1)) and _dense(torch.zeros(0, 3))
    assert _dense(torch.zeros(3, 1, 4)[:, :, :]) and _dense(torch.zeros(()))
    assert not _dense(t[:, ::2]) and not _dense(t[:, :, :3]) and not _dense(torch.zeros(3).expand(2, 3))


def test_layer_norm_entry_points_refuse():
    h = _lib.lib()
    fwd, bwd = h.m3d_layer_norm_fwd, h.m3d_layer_norm_bwd
    assert fwd(None, 8, None, None, 4, 8, 0, 0, 1e-5, 1.0, None, None, None, None) == -1
    assert fwd(P, 8, None, None, -1, 8, 0, 0, 1e-5, 1.0, P, None, None, None) == -1
    assert fwd(P, 8, None, None, 4, 0, 0, 0, 1e-5, 1.0, P, None, None, None) == -1
    assert fwd(P, 8, None, None, 4, 8, 3, 0, 1e-5, 1.0, P, None, None, None) == -1  # type
    assert fwd(P, 8, P, None, 4, 8, 0, 7, 1e-5, 1.0, P, None, None, None) == -1
    assert fwd(P + 2, 8, None, None, 4, 8, 0, 0, 1e-5, 1.0, P, None, None, None) == -1  # not aligned to its element
    assert fwd(P, 8, None, None, 4, 8, 0, 0, -1.0, 1.0, P, None, None, None) == -1
    assert fwd(P, 8, None, None, 4, 8, 0, 0, 1e-5, 1.0, P, P, None, None) == -1  # statistics: both or neither
    assert fwd(P, 8, None, None, 0, 8, 0, 0, 1e-5, 1.0, P, None, None, None) == 0  # no rows: nothing to do
    assert bwd(P, 8, P, 8, P, P, None, P, 4, 8, 0, 0, 1.0, P, P, P, P, None) == -1  # no statistics
    assert bwd(P, 8, P, 8, P, P, P, P, 4, 8, 0, 0, 1.0, P, P, P, None, None) == -1  # no workspace
    assert bwd(P, 8, P + 1, 8, P, P, P, P, 4, 8, 1, 0, 1.0, P, P, P, P, None) == -1
    assert bwd(P, 8, P, 8, P, P, P, P, 0, 8, 0, 0, 1.0, P, None, None, None, None) == 0
    size = h.m3d_layer_norm_bwd_workspace_bytes
    assert size(0, 8, 0) == 0 and size(10, 0, 0) == 0 and size(10, 8, 5) == 0
    assert size(1, 64, 0) == 2 * 64 * 4  # one workgroup, one row of partial sums


def _arrays(ptrs, numel, types):
    a = array("Q", ptrs), array("q", numel), array("i", types)
    return a, [t.buffer_info()[0] for t in a]


def test_many_tensor_entry_points_refuse():
    h = _lib.lib()
    nparts = ctypes.c_int32(0)
    at = ctypes.addressof(nparts)
    for ptrs, numel, types in (([P], [-1], [0]), ([P], [4], [3]), ([P + 2], [4], [0]), ([P + 1], [4], [1])):
        keep, (a, b, c) = _arrays(ptrs, numel, types)
        assert h.m3d_grad_norm(a, b, c, 1, P, at, None) == -1
        assert h.m3d_clip_grads(a, b, c, 1, P, 1, 1.0, P, None) == -1
    keep, (a, b, c) = _arrays([P], [4], [0])
    assert h.m3d_grad_norm(a, b, c, 1, None, at, None) == -1
    assert h.m3d_grad_norm(a, b, c, 1, P, None, None) == -1
    assert h.m3d_grad_norm(None, b, c, 1, P, at, None) == -1
    assert h.m3d_grad_norm(a, b, c, -1, P, at, None) == -1
    assert h.m3d_clip_grads(a, b, c, 1, P, 0, 1.0, P, None) == -1
    assert h.m3d_clip_grads(a, b, c, 1, P, 1 << 20, 1.0, P, None) == -1
    assert h.m3d_clip_grads(a, b, c, 1, P, 1, float("nan"), P, None) == -1
    keep2, (a2, b2, c2) = _arrays([P, P], [1 << 39, 1 << 39 | 1], [0, 0])
    assert h.m3d_grad_norm(a2, b2, c2, 2, P, at, None) == -2  # more elements than block numbers

    def step(**kw):
        args = dict(params=a, grads=a, numel=b, types=c, count=1, state_bits=32, exp_avg=P, exp_avg_sq=P, scale_avg=P, scale_avg_sq=P, state=P,
                    missed=P, parts=None, nparts=0, max_norm=0.0, norm_out=None, lr_dev=None, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
                    weight_decay=0.0)
        s = _lib.M3DAdamW(**{**args, **kw})
        return h.m3d_adamw_step(ctypes.addressof(s), None)

    assert h.m3d_adamw_step(None, None) == -1
    keep3, (none, _, _) = _arrays([0], [4], [0])
    for kw in ({"params": none}, {"exp_avg": None}, {"exp_avg_sq": P + 4}, {"state": None}, {"missed": None}, {"beta1": 1.0}, {"beta2": -0.5},
               {"state_bits": 8, "scale_avg": None}, {"parts": P, "nparts": 0}, {"parts": P, "nparts": 4, "max_norm": -1.0},
               {"eps": -1.0}, {"eps": float("nan")}, {"state_bits": 8, "eps": 0.0}):
        assert step(**kw) == -1, kw
    assert step(state_bits=16) == -2
    assert h.m3d_moments_decode(None, P, P, P, P, P, 1, None) == -1 and h.m3d_moments_decode(P, P, P, P, P, P + 4, 1, None) == -1
    assert h.m3d_moments_encode(P, P, P + 1, P, P, P, 1, None) == -1 and h.m3d_moments_encode(P, P, P, P, P, P, -1, None) == -1
    assert h.m3d_moments_decode(None, None, None, None, None, None, 0, None) == 0


def test_pointnet2_norm_choice():
    net = myria3d_amd.HipPointNet2(9, 6, norm="layer")
    names = set(net.state_dict())
    assert "sa1.nn.norms.0.module.weight" in names and not any("running" in n for n in names)
    assert {n for n, _ in net.named_parameters()} == {n for n, _ in myria3d_amd.HipPointNet2(9, 6).named_parameters()}
    with pytest.raises(ValueError):
        myria3d_amd.HipPointNet2(9, 6, norm="group")
