"""Network building blocks of the tracker's host-side modules.

Restates the reference's code/models/submodules.py (color_normalize 20-23,
convLayer 25-39, convLayer1d 41-55, fcLayer 57-61, initialize_weights 63-78)
so that modules built from them carry the reference's state_dict keys:
a block is nn.Sequential(conv[, batchnorm], ELU) -> keys `<name>.0.weight`,
`<name>.1.running_mean`, ...  A block may have group normalisation instead (norm='group'), whose
statistics do not depend on the batch: the same in training and in eval mode, at one pair a batch too.
"""
import math

import torch
import torch.nn as nn
from torch.nn import init
from torch.nn.modules import module as _nn_module

from .. import _native as N
from .. import ic
from .. import norm as gn
from .. import torch_ops  # noqa: F401  (registers the dpft:: ops torch.compile traces)

_RGB_MEAN = (0.4914, 0.4822, 0.4465)
_RGB_STD = (0.2023, 0.1994, 0.2010)


_NORM_CONSTS = {}


def color_normalize(color):
    """Per-channel (x - mean) / std of an RGB batch [B,3,H,W] (submodules.py:20-23).
    The constants are copied to the device once per (device, dtype): a host-to-device
    copy per call would also make forward impossible to capture in a HIP graph."""
    key = (color.device, color.dtype)
    if key not in _NORM_CONSTS:
        _NORM_CONSTS[key] = (torch.tensor(_RGB_MEAN, dtype=color.dtype, device=color.device).view(1, 3, 1, 1),
                             torch.tensor(_RGB_STD, dtype=color.dtype, device=color.device).view(1, 3, 1, 1))
    mean, std = _NORM_CONSTS[key]
    return (color - mean) / std


def _padding(kernel_size, dilation):
    # the reference's "same" padding formula (kept literally: it is not k//2*d for every d)
    return (kernel_size - 1) // 2 + dilation - 1


def _listened(m):
    """True where calling module m does more than its class's forward: hooks of its own or of every module (pruning,
    weight norm and spectral norm rebuild the weight in one), or a function put in forward's place."""
    return bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks
                or "forward" in m.__dict__ or _nn_module._has_any_global_hook())


class ConvBlock(nn.Sequential):
    """conv [-> batchnorm] -> ELU, an nn.Sequential (the reference's state_dict keys).
    In eval mode on the GPU, outside autograd, the batchnorm and the ELU of a 2-D block
    run as one in-place pass over the conv output (`ic.bn_elu_`, dpft_bn_elu) instead of
    two elementwise kernels; otherwise, or for a layout the kernel does not take, the
    modules run in turn.
    With a GroupNorm, a channels_last map (fp32, bf16, fp16) on the GPU goes through `norm.group_norm_act`, in
    training too; with `act_checkpoint` the backward pass then keeps the conv's input and output
    in 8 bits (`norm.conv2d`, `group_norm_act(checkpoint=True)`): 2 bytes a value, not 8.
    A module with hooks is called, and what it would have kept in 8 bits is kept in full."""

    act_checkpoint = False

    def _group(self, x):
        return (len(self) == 3 and isinstance(self[0], nn.Conv2d) and type(self[1]) is nn.GroupNorm
                and type(self[2]) is nn.ELU and self[2].alpha == 1.0 and x.is_cuda)

    def _group_conv(self, x):
        c = self[0]
        if (self.act_checkpoint and torch.is_grad_enabled() and type(c) is nn.Conv2d and c.padding_mode == 'zeros'
                and not isinstance(c.padding, str) and x.dim() == 4 and x.dtype in N.TYPES and not _listened(c)):
            return gn.conv2d(x, c.weight, c.bias, c.stride, c.padding, c.dilation, c.groups)
        return c(x)

    def _group_epilogue(self, y, packed=False):
        n = self[1]
        if (y.dim() != 4 or y.dtype not in N.TYPES or not y.is_contiguous(memory_format=torch.channels_last)
                or _listened(n) or _listened(self[2])):
            return self[2](n(y)).to(y.dtype)  # (autocast runs torch's group norm in fp32; the kernels keep y's type)
        return gn.group_norm_act(y, n.num_groups, n.weight, n.bias, n.eps, "elu", packed=packed,
                                 checkpoint=self.act_checkpoint)

    def _fusable(self, x):
        return (len(self) == 3 and isinstance(self[1], nn.BatchNorm2d) and isinstance(self[2], nn.ELU)
                and self[2].alpha == 1.0 and not self.training and x.is_cuda and not torch.is_grad_enabled())

    def forward_packed(self, x):
        """The block's output in the solver's channel-quad layout [B,C/4,H,W,4] when the
        epilogue can write it (dpft_bn_elu_pack: the batchnorm + ELU of a channels_last
        conv output stored out of place, no separate relayout pass); otherwise forward(x),
        [B,C,H,W].  Same values either way."""
        if self._group(x) and not torch.is_grad_enabled():
            y = self[0](x)
            return self._group_epilogue(y, packed=y.dtype == torch.float32 and y.dim() == 4 and y.shape[1] % 4 == 0)
        if self._fusable(x):
            y = self[0](x)
            if ic.bn_elu_pack_applies(y, self[1]):
                if torch.compiler.is_compiling():
                    return torch.ops.dpft.bn_elu_pack(y, torch_ops.bn_coeffs(self[1]))
                return ic.bn_elu_pack(y, self[1])
            return self._epilogue(y)
        return self.forward(x)

    def _epilogue(self, y):
        if torch.compiler.is_compiling():  # traced: the dpft::bn_elu_ op (torch_ops.py)
            if torch_ops.bn_elu_applies(y, self[1]):
                torch.ops.dpft.bn_elu_(y, torch_ops.bn_coeffs(self[1]))
                return y
        elif ic.bn_elu_(y, self[1]):
            return y
        return self[2](self[1](y))

    def forward(self, x):
        if self._group(x):
            return self._group_epilogue(self._group_conv(x))
        if self._fusable(x):
            return self._epilogue(self[0](x))
        return super().forward(x)


def _block(conv_cls, norm_fn, batch_norm, cin, cout, kernel_size, stride, dilation, bias):
    layers = [conv_cls(cin, cout, kernel_size=kernel_size, stride=stride,
                       padding=_padding(kernel_size, dilation), dilation=dilation,
                       bias=bias if batch_norm else True)]
    if batch_norm:
        layers.append(norm_fn(cout))
    layers.append(nn.ELU(inplace=True))
    return ConvBlock(*layers)


def group_norm(channels):
    """GroupNorm of 8 groups, or of the most that divide 8 and `channels`."""
    return nn.GroupNorm(math.gcd(8, channels), channels)


_NORMS = {'batch': nn.BatchNorm2d, 'group': group_norm}


def convLayer(batchNorm, in_planes, out_planes, kernel_size=3, stride=1, dilation=1, bias=False, norm='batch',
              act_checkpoint=False):
    """Conv2d [+ BatchNorm2d, or GroupNorm with norm='group'] + ELU; act_checkpoint (group norm only): ConvBlock, whose
    weights must be channels_last (with other maps the convolution's input alone is kept in 8 bits)."""
    if norm not in _NORMS:
        raise ValueError(f"norm must be one of {sorted(_NORMS)} (got {norm!r})")
    if act_checkpoint and (norm != 'group' or not batchNorm):
        raise ValueError("act_checkpoint needs norm='group'")
    block = _block(nn.Conv2d, _NORMS[norm], batchNorm, in_planes, out_planes, kernel_size, stride, dilation, bias)
    block.act_checkpoint = act_checkpoint
    return block


def convLayer1d(batchNorm, in_planes, out_planes, kernel_size=3, stride=1, dilation=1, bias=False):
    """Conv1d [+ BatchNorm1d] + ELU."""
    return _block(nn.Conv1d, nn.BatchNorm1d, batchNorm, in_planes, out_planes, kernel_size, stride, dilation, bias)


def fcLayer(in_planes, out_planes, bias=True):
    """Linear + ReLU."""
    return nn.Sequential(nn.Linear(in_planes, out_planes, bias), nn.ReLU(inplace=True))


def initialize_weights(modules, method='xavier'):
    """Xavier / Kaiming-uniform init of the Conv2d / ConvTranspose2d among `modules`
    (their direct iteration, as the reference does), zero biases."""
    for m in modules:
        if isinstance(m, (nn.Conv2d, nn.ConvTranspose2d)):
            if m.bias is not None:
                m.bias.data.zero_()
            if method == 'xavier':
                init.xavier_uniform_(m.weight)
            elif method == 'kaiming':
                init.kaiming_uniform_(m.weight)
