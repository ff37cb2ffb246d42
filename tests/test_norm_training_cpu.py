"""Training from 8-bit checkpoints on the CPU, with torch's own convolution gradients: norm.conv2d's function and the
encoder's blocks, the device operators replaced by their plain forms (norm_oracle).  What is under test is what this
package hands from the forward to the backward pass."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import norm_oracle as O
from deep_prob_feature_track_amd import norm
from deep_prob_feature_track_amd.models import submodules
from deep_prob_feature_track_amd.models.algorithms import FeaturePyramid

ARGS = [((1, 1), (0, 0), (1, 1), 1, 1), ((2, 1), (1, 2), (1, 2), 1, 3), ((1, 1), (2, 2), (2, 2), 4, 3)]


def _in_memory_order(x):
    """x's values as they lie in memory, and a function that puts such values back into x's shape and strides."""
    order = sorted(range(x.dim()), key=lambda d: -x.stride(d))
    p = x.permute(order)
    assert p.is_contiguous()
    back = [order.index(d) for d in range(x.dim())]
    return p.reshape(-1), lambda flat: flat.view(p.shape).permute(back)


def _restored(x):
    flat, put = _in_memory_order(x.detach())
    return put(O.through_8_bits(flat.double())[0].to(x.dtype))


@pytest.fixture
def plain(monkeypatch):
    """act_checkpoint and act_restore by their definition."""
    def act_checkpoint(x):
        x = norm._dense(x.detach())
        flat, codes = O.through_8_bits(_in_memory_order(x)[0].double())
        step = ((codes + (1023 - 133)) << 52).view(torch.float64).repeat_interleave(32)[:flat.numel()]
        return norm.ActCheckpoint((flat / step).to(torch.int8), codes.to(torch.uint8), x.shape, x.stride(), x.dtype)

    def act_restore(c, dtype=None):
        step = ((c.scale.long() + (1023 - 133)) << 52).view(torch.float64).repeat_interleave(32)[:c.q.numel()]
        out = torch.empty_strided(c.shape, c.stride, dtype=c.dtype if dtype is None else dtype)
        return _in_memory_order(out)[1]((c.q.double() * step).to(out.dtype))
    monkeypatch.setattr(norm, "act_checkpoint", act_checkpoint)
    monkeypatch.setattr(norm, "act_restore", act_restore)


@pytest.mark.parametrize("layout", ["nchw", "channels_last", "slice"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("stride,padding,dilation,groups,k", ARGS)
def test_conv2d_gradients(plain, layout, bias, stride, padding, dilation, groups, k):
    """y and dx are the convolution's own; dw and db those at the restored input."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(2, 8, 12, 15, generator=g)
    if layout == "slice":
        x = torch.randn(2, 8, 14, 16, generator=g)[:, :, 1:13, :15]
    x = x.contiguous(memory_format=torch.channels_last) if layout == "channels_last" else x
    w = 0.2 * torch.randn(12, 8 // groups, k, k, generator=g)
    b = torch.randn(12, generator=g) if bias else None
    ins = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = norm._Conv2dCheckpoint.apply(*(ins + [None] if not bias else ins), list(stride), list(padding), list(dilation), groups)
    dy = torch.randn(y.shape, generator=g)
    got = torch.autograd.grad(y, ins, dy)

    def plainly(x):
        v = [t.detach().double().requires_grad_(True) for t in ((x, w, b) if bias else (x, w))]
        out = F.conv2d(*(v if bias else v + [None]), stride, padding, dilation, groups)
        return out, torch.autograd.grad(out, v, dy.double())
    want_y, (want_dx, *_) = plainly(x)
    _, (_, *want_params) = plainly(_restored(x if layout != "slice" else x.contiguous()))
    # y: 8 k k / groups products, dx: 12 k k / groups, dw and db: 2 x 12 x 15 and fewer, each in some order
    scale = {"y": 8 * k * k, "dx": 12 * k * k, "dw": 360, "db": 360}
    mag_y = F.conv2d(x.abs().double(), w.abs().double(), b.abs().double() if bias else None, stride, padding, dilation, groups)
    assert ((y.double() - want_y).abs() <= scale["y"] * O.U * mag_y).all()
    assert ((got[0].double() - want_dx).abs() <= scale["dx"] * O.U * w.abs().sum().double() * dy.abs().max()).all()
    top = dy.abs().sum().double()
    for name, a, r in zip(("dw", "db"), got[1:], want_params):
        assert ((a.double() - r).abs() <= scale[name] * O.U * top * max(1.0, float(x.abs().max()))).all(), name
    # a value's rounding to 8 bits shows, so that dw is not the plain one
    assert (want_params[0] - plainly(x)[1][1]).abs().max() > 100 * 360 * O.U


def test_conv2d_keeps_bytes_and_may_run_twice(plain):
    x = torch.randn(2, 8, 6, 7).requires_grad_(True)
    w = torch.randn(4, 8, 1, 1).requires_grad_(True)
    y = norm._Conv2dCheckpoint.apply(x, w, None, [1, 1], [0, 0], [1, 1], 1)
    kept = [t for t in y.grad_fn.saved_tensors if t is not None]
    assert sorted(str(t.dtype) for t in kept) == ["torch.float32", "torch.int8", "torch.uint8"]  # the weight, q, scale
    one = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    two = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    assert all(torch.equal(u, v) for u, v in zip(one, two))
    g, = torch.autograd.grad(y.sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.no_grad():  # the input may change after the forward pass: what was kept is its copy
        x.mul_(2)
    assert torch.equal(torch.autograd.grad(y.sum(), w)[0], one[1])


class _NormFrom8Bits(torch.autograd.Function):
    """act(group_norm(x)) with the gradients at the restored x and x's own statistics, from the formulas."""

    @staticmethod
    def forward(ctx, x, groups, weight, bias, eps):
        ctx.save_for_backward(x, weight, bias)
        ctx.groups, ctx.eps = groups, eps
        return O.Reference(x, groups, weight, bias, eps, "elu").y.to(x.dtype)

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        r = O.Reference(x, ctx.groups, weight, bias, ctx.eps, "elu", dy, checkpoint=True)
        return r.dx.to(x.dtype), None, r.dweight.to(weight.dtype), r.dbias.to(bias.dtype), None


def test_encoder_training_step(plain, monkeypatch):
    """A training step of the whole encoder through its device path: all 20 blocks keep their activations in 8 bits,
    the outputs are the plain encoder's, and so are the gradients but for the stored values' rounding.  Each is off by
    at most 1/128 of its block's largest (rms 1/222 of it, and that is about 4 times a value's own rms: 2 % of it);
    twenty blocks deep, independent: sqrt(20) x 2 % = 9 %, and as much again for the weights' own factors."""
    convs, norms = [], []

    def conv2d(x, weight, bias, *conv):
        convs.append(x.shape)
        return norm._Conv2dCheckpoint.apply(x, weight, bias, *(list(c) if isinstance(c, tuple) else c for c in conv))

    def group_norm_act(y, groups, weight, bias, eps, act, packed=False, checkpoint=False):
        assert act == "elu" and checkpoint and not packed
        norms.append(y.shape)
        return _NormFrom8Bits.apply(y, groups, weight, bias, eps)
    torch.manual_seed(5)
    enc = FeaturePyramid(D=8, w_uncertainty="laplacian", feature_channel=8, feature_extract="conv", uncertainty_channel=1,
                         norm="group", act_checkpoint=True).to(memory_format=torch.channels_last).train()
    with torch.no_grad():
        for m in enc.modules():
            if isinstance(m, nn.GroupNorm):
                m.weight.add_(0.3 * torch.randn_like(m.weight))
                m.bias.add_(0.3 * torch.randn_like(m.bias))
    x = torch.randn(2, 8, 48, 64).contiguous(memory_format=torch.channels_last)

    def step():
        f, s, _ = enc(x)
        loss = sum((t * t).mean() for t in f) + sum(t.log().square().mean() for t in s)
        return [t.detach() for t in f + s], torch.autograd.grad(loss, list(enc.parameters()))
    outs, grads = step()
    monkeypatch.setattr(submodules.gn, "group_norm_act", group_norm_act)
    monkeypatch.setattr(submodules.gn, "conv2d", conv2d)
    monkeypatch.setattr(submodules.ConvBlock, "_group", lambda self, x: type(self[1]) is nn.GroupNorm)
    outs8, grads8 = step()
    assert len(convs) == len(norms) == 20
    for a, b in zip(outs8, outs):  # (the bound of test_norm_encoder.py: twenty blocks of at most 1152 products)
        assert (a - b).abs().max() <= 20 * 1152 * O.U * b.abs().max()
    for a, b in zip(grads8, grads):
        assert torch.isfinite(a).all() and (a - b).norm() <= 0.18 * b.norm() + 1e-6
    assert any(not torch.equal(a, b) for a, b in zip(grads8, grads))
