"""Group normalisation with an activation, and activation checkpoints in 8 bits (device tensors).

`group_norm_act` is an encoder block's epilogue (conv -> norm -> activation) whose statistics come
from the sample itself: the same in training and in eval mode, at any batch size.  `act_checkpoint`
/ `act_restore` keep an activation in 8 bits (a shared power-of-two step for each 32 values), and
`conv2d` keeps its input that way for its weight gradient.  With `checkpoint=True` a block's
backward pass needs 2 bytes a value of its two activations, not 8.

Thin marshalling over libdpft_ic.so, as ic.py: they validate shapes, hand device pointers and the
current stream to the C ABI and never synchronise; every call has a workspace of its own, so calls
on several streams, and captured graphs, share nothing.  CPU tensors raise: the modules of
models/submodules.py take the torch path for them.
"""
import contextlib
import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .ic import _eager_only

BLOCK = 32  # values that share a step in a checkpoint


def _check_device(x, what):
    if x.dtype not in N.TYPES:
        raise TypeError(f"{what}: float32, bfloat16 or float16 (got {x.dtype})")
    if not x.is_cuda:
        raise RuntimeError(f"{what} needs a device tensor; there is no CPU fallback")


def _check_param(p, name, x):
    if p.dim() != 1 or p.shape[0] != x.shape[1]:
        raise ValueError(f"{name} must hold one value per channel ({x.shape[1]}), got {tuple(p.shape)}")
    if p.dtype not in N.TYPES:
        raise TypeError(f"{name}: float32, bfloat16 or float16 (got {p.dtype})")
    if p.device != x.device:
        raise ValueError(f"{name} is on {p.device}, expected {x.device}")


def _nhwc(x):
    """x [N,C,H,W] stored channels_last and 16-byte aligned (a copy where it is not)."""
    if not x.is_contiguous(memory_format=torch.channels_last):
        x = x.contiguous(memory_format=torch.channels_last)
    if x.data_ptr() % 16:
        x = x.clone(memory_format=torch.channels_last)
    return x


def _empty_nhwc(x):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device, memory_format=torch.channels_last)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _on(device):
    """Launches go to the tensors' device, whichever is the current one."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


@functools.lru_cache(maxsize=4096)
def _plan(shape, groups, act, x_type, param_type, flags, eps):
    """(descriptor, its address, workspace bytes) of a call's sizes and types."""
    B, C, H, W = shape
    desc = N.GroupNorm(H * W, B, C, groups, N.ACTS[act], x_type, param_type, flags, eps)
    ref = ctypes.byref(desc)
    nbytes = N.lib().dpft_group_norm_workspace_size(ref)
    if nbytes == 0:
        N.check(-1, "dpft_group_norm_workspace_size")
    return desc, ref, nbytes


def _call(x, groups, weight, bias, eps, act, flags=0):
    """(descriptor's address, workspace bytes, workspace) for x's sizes; a workspace of the call's own."""
    p = weight if weight is not None else bias
    _, ref, nbytes = _plan(tuple(x.shape), groups, act, N.TYPES[x.dtype], 0 if p is None else N.TYPES[p.dtype], flags, eps)
    return ref, nbytes, torch.empty(nbytes, dtype=torch.uint8, device=x.device)


class ActCheckpoint:
    """An activation in 8 bits: `q` [n] int8 and `scale` [ceil(n / 32)] uint8 in memory order, and the
    shape, strides and dtype it is restored with (include/dpft_ic.h, dpft_act_checkpoint)."""

    __slots__ = ("q", "scale", "shape", "stride", "dtype")

    def __init__(self, q, scale, shape, stride, dtype):
        self.q, self.scale, self.shape, self.stride, self.dtype = q, scale, shape, stride, dtype

    def nbytes(self):
        return self.q.numel() + self.scale.numel()


def _checkpoint_buffers(n, device):
    return (torch.empty(n, dtype=torch.int8, device=device),
            torch.empty((n + BLOCK - 1) // BLOCK, dtype=torch.uint8, device=device))


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
    127 steps clamp the largest).  A block with an infinity or a NaN restores as NaN."""
    _check_device(x, "act_checkpoint")
    x = _dense(x.detach())
    n = x.numel()
    q, scale = _checkpoint_buffers(n, x.device)
    c = ActCheckpoint(q, scale, x.shape, x.stride(), x.dtype)
    if n:
        if x.data_ptr() % 16:
            x = x.clone(memory_format=torch.preserve_format)
        with _on(x.device):
            N.check(N.lib().dpft_act_checkpoint(_ptr(x), N.TYPES[x.dtype], n, _ptr(q), _ptr(scale), _stream(x.device)),
                    "dpft_act_checkpoint")
    return c


@_eager_only
def act_restore(c, dtype=None):
    """The values of an ActCheckpoint, in its own dtype or in `dtype` (exact in fp32 and bf16; rounded
    once in fp16 where its range ends)."""
    dtype = c.dtype if dtype is None else dtype
    if dtype not in N.TYPES:
        raise TypeError(f"act_restore: float32, bfloat16 or float16 (got {dtype})")
    out = torch.empty_strided(c.shape, c.stride, dtype=dtype, device=c.q.device)
    if out.numel():
        with _on(out.device):
            N.check(N.lib().dpft_act_restore(_ptr(c.q), _ptr(c.scale), c.q.numel(), _ptr(out), N.TYPES[dtype],
                                             _stream(out.device)), "dpft_act_restore")
    return out


def _forward(x, groups, weight, bias, eps, act, packed, stats, checkpoint):
    """-> y, statistics [2,N,groups], q, scale (None where not asked for); x channels_last."""
    B, C, H, W = x.shape
    if packed:
        y = torch.empty(B, C // 4, H, W, 4, dtype=x.dtype, device=x.device)
    else:
        y = _empty_nhwc(x)
    stat = torch.empty(2, B, groups, dtype=torch.float32, device=x.device) if stats else None
    q, scale = _checkpoint_buffers(x.numel(), x.device) if checkpoint else (None, None)
    if x.numel():
        with _on(x.device):
            ref, nbytes, ws = _call(x, groups, weight, bias, eps, act, N.GN_PACKED if packed else 0)
            mean = _ptr(stat)
            rc = N.lib().dpft_group_norm_act(ref, x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), mean,
                                             mean + 4 * B * groups if stats else None, _ptr(q), _ptr(scale),
                                             ws.data_ptr(), nbytes, _stream(x.device))
            if rc:
                N.check(rc, "dpft_group_norm_act")
    return y, stat, q, scale


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, checkpoint):
        x = _nhwc(x)
        w = weight if weight is None else weight.contiguous()
        b = bias if bias is None else bias.contiguous()
        y, stat, q, scale = _forward(x, groups, w, b, eps, act, False, True, checkpoint)
        ctx.args = (groups, eps, act)
        ctx.save_for_backward(None if checkpoint else x, q, scale, w, b, stat)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, q, scale, w, b, stat = ctx.saved_tensors
        groups, eps, act = ctx.args
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = _nhwc(dy)
        dx = _empty_nhwc(dy) if need_x else None
        dw = torch.empty_like(w) if need_w else None
        db = torch.empty_like(b) if need_b else None
        if dy.numel() == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        else:
            with _on(dy.device):
                ref, nbytes, ws = _call(dy, groups, w, b, eps, act)
                mean = stat.data_ptr()
                rc = N.lib().dpft_group_norm_act_backward(
                    ref, dy.data_ptr(), _ptr(x), _ptr(q), _ptr(scale), _ptr(w), _ptr(b), mean,
                    mean + 4 * dy.shape[0] * groups, _ptr(dx), _ptr(dw), _ptr(db), ws.data_ptr(), nbytes,
                    _stream(dy.device))
                if rc:
                    N.check(rc, "dpft_group_norm_act_backward")
        return dx, dw, db, None, None, None, None


@_eager_only
def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="elu", packed=False, checkpoint=False):
    """act(group_norm(x)) of a map [N,C,H,W] in fp32, bf16 or fp16, channels_last (other layouts are
    copied; the result is channels_last), differentiable once in x, weight and bias.

    groups divides C; weight / bias [C] (fp32 or another float type, both alike; None: 1 / 0); act
    'none', 'relu', 'elu' or 'silu'.
    packed=True (inference, fp32, C % 4 == 0): the solver's channel-quad layout [N,C/4,H,W,4].
    checkpoint=True: the backward pass keeps x as an 8-bit checkpoint (act_checkpoint) instead of x,
    written by the forward launch; y is that of x, the gradients are those at the restored x with x's
    own statistics."""
    if x.dim() != 4:
        raise ValueError(f"group_norm_act needs a map [N,C,H,W], got {tuple(x.shape)}")
    if act not in N.ACTS:
        raise ValueError(f"act must be one of {sorted(N.ACTS)} (got {act!r})")
    C = x.shape[1]
    if groups < 1 or C % groups or C == 0:
        raise ValueError(f"groups={groups} does not divide C={C}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative (got {eps})")
    if weight is not None:
        _check_param(weight, "weight", x)
    if bias is not None:
        _check_param(bias, "bias", x)
        if weight is not None and weight.dtype != bias.dtype:
            raise TypeError(f"weight and bias must have one dtype (got {weight.dtype}, {bias.dtype})")
    grad = torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                        or (bias is not None and bias.requires_grad))
    if packed:
        if grad:
            raise RuntimeError("packed=True is the solver's input at inference: it has no backward")
        if x.dtype != torch.float32 or C % 4:
            raise ValueError(f"packed=True needs fp32 and C % 4 == 0, got {x.dtype} {tuple(x.shape)}")
    _check_device(x, "group_norm_act")
    if grad:
        return _GroupNormAct.apply(x, weight, bias, groups, eps, act, checkpoint)
    return _forward(_nhwc(x), groups, weight if weight is None else weight.contiguous(),
                    bias if bias is None else bias.contiguous(), eps, act, packed, False, False)[0]


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
        dx, dw, db = torch.ops.aten.convolution_backward(dy, x, weight, ctx.bias_sizes, stride, padding, dilation,
                                                         False, [0, 0], groups, list(ctx.needs_input_grad[:3]))
        return dx, dw, db, None, None, None, None


def _pair(v):
    return [v, v] if isinstance(v, int) else list(v)


@_eager_only
def conv2d(x, weight, bias=None, stride=1, padding=0, dilation=1, groups=1):
    """torch.nn.functional.conv2d whose backward pass keeps x as an 8-bit checkpoint: the same y and
    gradient of x, the weight's gradient at the restored x.  Under autocast, in its dtype."""
    if isinstance(padding, str):
        raise ValueError(f"padding must be numbers (got {padding!r})")
    _check_device(x, "conv2d")
    args = (_pair(stride), _pair(padding), _pair(dilation), groups)
    if not (torch.is_grad_enabled() and weight.requires_grad):  # the backward pass does not read x
        return torch.nn.functional.conv2d(x, weight, bias, *args)
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(dt), weight.to(dt), None if bias is None else bias.to(dt)
        with torch.autocast("cuda", enabled=False):
            return _Conv2dCheckpoint.apply(x, weight, bias, *args)
    return _Conv2dCheckpoint.apply(x, weight, bias, *args)
