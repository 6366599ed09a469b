"""CPU: refusals of the training-side operators that come before anything is written."""
import pytest
import torch

import myria3d_amd


def test_clip_refuses_a_gradient_that_cannot_be_scaled_in_place():
    """Before the others are scaled, and not from within the copy back."""
    p, q = torch.zeros(3, 4, requires_grad=True), torch.zeros(3, 4, requires_grad=True)
    p.grad = torch.ones(3, 4)
    for spread in (torch.ones(1, 4).expand(3, 4), torch.ones(()).expand(3, 4)):
        q.grad = spread
        with pytest.raises(RuntimeError, match="share memory"):
            myria3d_amd.clip_grad_norm_([p, q], 0.5)
    q = torch.zeros(1, 4, requires_grad=True)
    q.grad = torch.ones(4, 1).t()[:, ::1].as_strided((1, 4), (0, 1))  # one row: its stride says nothing
    with pytest.raises(RuntimeError, match="MI355X"):
        myria3d_amd.clip_grad_norm_([p, q], 0.5)
