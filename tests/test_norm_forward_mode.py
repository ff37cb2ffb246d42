"""Forward-mode derivatives of the normalisation operators: there are none, so that an input with a tangent is
refused in every way of calling (meta tensors: nothing here needs a device)."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from deep_prob_feature_track_amd import _native as N
from deep_prob_feature_track_amd import norm

MATCH = "forward-mode"


def _inputs():
    return torch.zeros(2, 8, 4, 4, device="meta"), torch.ones(8, device="meta"), torch.zeros(8, device="meta")


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
@pytest.mark.parametrize("grad_enabled", [False, True])
@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_a_tangent_is_refused(which, grad_enabled, requires_grad, packed):
    x, w, b = _inputs()
    with fwAD.dual_level(), torch.set_grad_enabled(grad_enabled):
        args = {"x": x, "weight": w, "bias": b}
        args[which] = fwAD.make_dual(args[which].requires_grad_(requires_grad), torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match=MATCH):
            norm.group_norm_act(args["x"], 4, args["weight"], args["bias"], packed=packed)


def test_function_transforms_are_refused():
    x, w, b = _inputs()

    def f(t):
        return norm.group_norm_act(t, 4, w, b)
    with pytest.raises(NotImplementedError, match=MATCH):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with pytest.raises(NotImplementedError, match=MATCH):
        torch.func.jvp(lambda v: norm.group_norm_act(x, 4, v), (w,), (w,))
    with pytest.raises(NotImplementedError, match=MATCH):
        torch.func.jacfwd(f)(x)
    for transform in (torch.func.jacrev(f), torch.func.grad(lambda t: f(t).sum())):
        with pytest.raises(RuntimeError):
            transform(x)


def test_the_operators_refuse_a_tangent():
    ops = N.torch_ops()
    x, w, b = _inputs()
    none, stat = torch.empty(0, device="meta"), torch.empty(2, 2, 4, device="meta")
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match=MATCH):
            ops.group_norm_act_forward(d, 4, w, b, 1e-5, 2, False, True, False)
        for dy, xs in ((d, x), (x, d)):
            with pytest.raises(NotImplementedError, match=MATCH):
                ops.group_norm_act_backward(dy, xs, none, none, w, b, stat, 4, 1e-5, 2, True, True, True)
        y = norm.group_norm_act(x.clone().requires_grad_(True), 4, w, b)  # a gradient that carries a tangent
        with pytest.raises(NotImplementedError, match=MATCH):
            y.backward(fwAD.make_dual(torch.zeros_like(x), x))


def test_without_a_tangent_a_dual_level_changes_nothing():
    x, w, b = _inputs()
    with fwAD.dual_level():
        assert norm.group_norm_act(x, 4, w, b).shape == x.shape
        y = norm.group_norm_act(x.requires_grad_(True), 4, w, b)
        dx, = torch.autograd.grad(y, x, torch.zeros_like(y))
        assert dx.shape == x.shape
