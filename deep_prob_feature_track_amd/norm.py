"""Group normalisation with an activation, and activation checkpoints in 8 bits (device tensors).

`group_norm_act` is an encoder block's epilogue (conv -> norm -> activation) whose statistics come
from the sample itself: the same in training and in eval mode, at any batch size.  `act_checkpoint`
/ `act_restore` keep an activation in 8 bits (a shared power-of-two step for each 32 values), and
`conv2d` keeps its input that way for its weight gradient.  With `checkpoint=True` a block's
backward pass needs 2 bytes a value of its two activations, not 8.

The operators are `torch.ops.dpft.*` of libdpft_torch.so over the C ABI (include/dpft_ic.h): they check
their arguments, launch on the current stream of the tensors' device and never synchronise; every call
has a workspace of its own, so that calls on several streams, and captured graphs, share nothing; they
trace under torch.compile.  CPU tensors raise: the modules of models/submodules.py take the torch path
for them.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .ic import _eager_only

BLOCK = 32  # values that share a step in a checkpoint

# loaded with the module, so that nothing is left to a traced call.  A library that is missing or does not load (half
# written, stale, of another torch) does not end the import, which the CPU's and batch norm's users need too: every
# call then tries again and raises.
try:
    _ops = N.torch_ops()
except (OSError, RuntimeError, AttributeError):
    _ops = None


def _op(name):
    return getattr(_ops if _ops is not None else N.torch_ops(), name).default


class ActCheckpoint:
    """An activation in 8 bits: `q` [n] int8 and `scale` [ceil(n / 32)] uint8 in memory order, and the
    shape, strides and dtype it is restored with (include/dpft_ic.h, dpft_act_checkpoint)."""

    __slots__ = ("q", "scale", "shape", "stride", "dtype")

    def __init__(self, q, scale, shape, stride, dtype):
        self.q, self.scale, self.shape, self.stride, self.dtype = q, scale, shape, stride, dtype

    def nbytes(self):
        return self.q.numel() + self.scale.numel()


def _dense(x):
    """x without gaps or overlaps in memory, in its own order of dimensions (a copy where it has)."""
    expect = 1
    for size, stride in sorted(((s, st) for s, st in zip(x.shape, x.stride()) if s > 1), key=lambda a: a[1]):
        if stride != expect:
            return x.contiguous()
        expect *= size
    return x


@_eager_only
def act_checkpoint(x):
    """x (fp32, bf16 or fp16, any shape) in 8 bits -> ActCheckpoint.  Values go in blocks of 32 in
    memory order (a channels_last map: along its channels), each block with a step of 2^(E - 6) where
    2^E <= max |x| < 2^(E + 1): off by at most half a step, max |x| / 128 and less (a whole step where
    127 steps clamp the largest).  A block with an infinity or a NaN restores as NaN.
    Outside autograd: no gradient and no tangent goes through.  A traced call runs it eagerly (a graph break;
    fullgraph=True raises), as act_restore and conv2d."""
    x = _dense(x.detach())
    q, scale = _op("act_checkpoint")(x)
    return ActCheckpoint(q, scale, x.shape, x.stride(), x.dtype)


@_eager_only
def act_restore(c, dtype=None):
    """The values of an ActCheckpoint, in its own dtype or in `dtype` (exact in fp32 and bf16; rounded
    once in fp16 where its range ends)."""
    return _op("act_restore")(c.q, c.scale, c.shape, c.stride, c.dtype if dtype is None else dtype)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="elu", packed=False, checkpoint=False):
    """act(group_norm(x)) of a map [N,C,H,W] in fp32, bf16 or fp16, channels_last (other layouts are
    copied; the result is channels_last), differentiable once in x, weight and bias by the backward pass.
    There is no forward-mode derivative: an input that carries a tangent raises NotImplementedError, and of
    torch.func's transforms only vmap runs it (a call for each sample).

    groups divides C; weight / bias [C] (fp32 or another float type, both alike; None: 1 / 0); act
    'none', 'relu', 'elu' or 'silu'.
    packed=True (inference, fp32, C % 4 == 0): the solver's channel-quad layout [N,C/4,H,W,4].
    checkpoint=True: the backward pass keeps x as an 8-bit checkpoint (act_checkpoint) instead of x,
    written by the forward pass; y is that of x, the gradients are those at the restored x with x's
    own statistics."""
    code = N.ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {sorted(N.ACTS)} (got {act!r})")
    return _op("group_norm_act")(x, groups, weight, bias, eps, code, packed, checkpoint)


_convolution_backward = torch.ops.aten.convolution_backward


class _Conv2dCheckpoint(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, stride, padding, dilation, groups):
        c = act_checkpoint(x)
        ctx.save_for_backward(weight, c.q, c.scale)
        ctx.layout = (c.shape, c.stride, c.dtype)
        ctx.conv = (stride, padding, dilation, groups)
        ctx.bias_sizes = None if bias is None else list(bias.shape)
        return torch.nn.functional.conv2d(x, weight, bias, stride, padding, dilation, groups)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, q, scale = ctx.saved_tensors
        stride, padding, dilation, groups = ctx.conv
        x = act_restore(ActCheckpoint(q, scale, *ctx.layout))
        dx, dw, db = _convolution_backward(dy, x, weight, ctx.bias_sizes, stride, padding, dilation, False, [0, 0], groups,
                                           list(ctx.needs_input_grad[:3]))
        return dx, dw, db, None, None, None, None


def _pair(v):
    return [v, v] if isinstance(v, int) else list(v)


@_eager_only
def conv2d(x, weight, bias=None, stride=1, padding=0, dilation=1, groups=1):
    """torch.nn.functional.conv2d whose backward pass keeps x as an 8-bit checkpoint: the same y and
    gradient of x, the weight's gradient at the restored x.  Under autocast, in its dtype.  Not covered by a running
    test with the device library's own convolution gradients (the CPU's are, and what the device's are handed)."""
    if isinstance(padding, str):
        raise ValueError(f"padding must be numbers (got {padding!r})")
    if not x.is_cuda:
        raise RuntimeError("conv2d needs a device tensor; there is no CPU fallback")
    if x.dim() != 4:
        raise ValueError(f"conv2d needs a map [N,C,H,W], got {tuple(x.shape)}")
    args = (_pair(stride), _pair(padding), _pair(dilation), groups)
    if not (torch.is_grad_enabled() and weight.requires_grad):  # the backward pass does not read x
        return torch.nn.functional.conv2d(x, weight, bias, *args)
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(dt), weight.to(dt), None if bias is None else bias.to(dt)
        with torch.autocast("cuda", enabled=False):
            return _Conv2dCheckpoint.apply(x, weight, bias, *args)
    return _Conv2dCheckpoint.apply(x, weight, bias, *args)
