"""The normalisation operators of the feature encoder: what a pass of each computes, reads and writes.

Kinds of case:
  infer       y = act(group_norm(x)), channels last, outside autograd
  packed      the same, stored in the solver's channel-quad layout [N,C/4,H,W,4]
  train       forward and backward: y and the gradients of x, weight and bias
  store8      an activation checkpoint in 8 bits and its restoration
  train8      forward and backward, where the forward keeps its input in 8 bits only

`run` computes a case from elementary torch operations, or (own = True) makes the calls that a
user makes of deep_prob_feature_track_amd.norm.  `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-5
BLOCK = 32  # values that share one scale in an 8-bit checkpoint
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _case(name, kind, n, c, h, w, groups, dtype="f32", act="elu"):
    return {"name": name, "kind": kind, "n": n, "c": c, "h": h, "w": w, "groups": groups, "dtype": dtype, "act": act}


def listed():
    """The encoder's maps (16 to 128 channels, 640x480 halved three times, 8 pairs in a call),
    the keyframe tracker's single small images (160x120), and an odd one."""
    return [
        # the coarsest map of one 160x120 image: a call that is all latency
        _case("infer_small", "infer", 1, 128, 15, 20, 8),
        # the second scale of 8 images of 640x480 under mixed precision
        _case("infer_half", "infer", 8, 64, 240, 320, 8, "bf16"),
        # the full-resolution backbone map of 8 images of 640x480
        _case("infer_large", "infer", 8, 32, 480, 640, 8),
        # a feature head of one 160x120 image and one of 8 images of 640x480, written as the solver reads them
        _case("packed_single", "packed", 1, 32, 120, 160, 8),
        _case("packed_heads", "packed", 8, 32, 240, 320, 8),
        # a training step's block on an odd crop, its groups narrower than a load
        _case("train_odd", "train", 3, 30, 61, 79, 5, "f16", "silu"),
        # the third scale of a training batch of 8 images of 640x480
        _case("train_third", "train", 8, 96, 120, 160, 8),
        # the second scale of both frames of 8 pairs under mixed precision
        _case("train_half", "train", 16, 64, 240, 320, 8, "bf16"),
        # checkpoints of a convolution's input: an odd one, and the full-resolution map of 8 images
        _case("store8_odd", "store8", 1, 13, 61, 79, 1, "f16"),
        _case("store8_large", "store8", 8, 32, 480, 640, 1),
        # a block of one 160x120 image, and the second scale of 8 images, trained from 8-bit checkpoints
        _case("train8_single", "train8", 1, 16, 120, 160, 8),
        _case("train8_second", "train8", 8, 64, 240, 320, 8),
    ]


def draw(rng):
    """Any kind and type, 1 to 16 images, 1 to 640 pixels a side, 1 to 512 channels in groups of
    1 to 64, up to the largest map above."""
    kind = rng.choice(["infer", "packed", "train", "store8", "train8"])
    dtype = "f32" if kind == "packed" else rng.choice(["f32", "bf16", "f16"])
    act = rng.choice(["elu", "silu", "none"] + (["relu"] if kind in ("infer", "packed") else []))
    while True:
        n = rng.choice([1, 2, 3, 4, 6, 8, 16])
        groups = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
        c = groups * rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64])
        h = int(round(math.exp(rng.uniform(0.0, math.log(480)))))
        w = int(round(math.exp(rng.uniform(0.0, math.log(640)))))
        if c > 512 or (kind == "packed" and c % 4) or n * c * h * w < 1000:
            continue
        if n * c * h * w > (20e6 if kind in ("train", "train8") else 39e6):
            continue
        return {"kind": kind, "n": n, "c": c, "h": h, "w": w, "groups": groups, "dtype": dtype, "act": act}


def prepare(case, seed):
    """A convolution's output as training leaves it: channels of unlike mean and spread, images of
    unlike brightness; the affine parameters near 1 and 0; a small gradient."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) & 0x7FFFFFFF)
    n, c, h, w = case["n"], case["c"], case["h"], case["w"]
    dt = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    x = normal(n, h, w, c)
    x = x.mul_(torch.exp(0.5 * normal(c))).add_(normal(c)).mul_(torch.exp(0.3 * normal(n, 1, 1, 1)))
    st = {"case": case, "x": x.to(dt).permute(0, 3, 1, 2)}
    if case["kind"] == "store8":
        return st
    st["weight"] = 1.0 + 0.3 * normal(c)
    st["bias"] = 0.3 * normal(c)
    if case["kind"] in ("train", "train8"):
        st["dy"] = (1e-2 * normal(n, h, w, c)).to(dt).permute(0, 3, 1, 2)
        for k in ("x", "weight", "bias"):
            st[k] = st[k].requires_grad_(True)
    return st


# ------------------------------------------------------------------ the framework's calls
def _run_own(st):
    from deep_prob_feature_track_amd import norm
    case = st["case"]
    kind, groups, act = case["kind"], case["groups"], case["act"]
    if kind == "store8":
        return norm.act_restore(norm.act_checkpoint(st["x"]))
    if kind in ("infer", "packed"):
        with torch.no_grad():
            return norm.group_norm_act(st["x"], groups, st["weight"], st["bias"], eps=EPS, act=act,
                                       packed=kind == "packed")
    y = norm.group_norm_act(st["x"], groups, st["weight"], st["bias"], eps=EPS, act=act, checkpoint=kind == "train8")
    dx, dw, db = torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


# ------------------------------------------------------------------ the plain form
def _act(z, act):
    if act == "elu":
        return torch.where(z > 0, z, torch.expm1(torch.clamp(z, max=0.0)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "relu":
        return torch.clamp(z, min=0.0)
    return z


def _act_slope(z, act):
    if act == "elu":
        return torch.exp(torch.clamp(z, max=0.0))
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _through_8_bits(flat):
    """Values in 8 bits by blocks of 32 in memory order, one power of two to a block: 2^(E - 6)
    with E the exponent of the block's largest magnitude, so that it comes to 64 .. 127 steps."""
    n = flat.numel()
    blocks = torch.nn.functional.pad(flat, (0, -n % BLOCK)).view(-1, BLOCK)
    top = blocks.abs().amax(1, keepdim=True)
    exponent = (top.view(torch.int32) >> 23).clamp(7, 254)
    finite = blocks.isfinite().all(1, keepdim=True)
    scale = ((exponent - 6) << 23).view(torch.float32)
    inverse = ((260 - exponent) << 23).view(torch.float32)
    q = torch.clamp(torch.round(blocks * inverse), -127, 127) * scale
    q = torch.where(finite, q, torch.full_like(q, float("nan")))
    return q.view(-1)[:n]


def _run_plain(st):
    case = st["case"]
    kind, groups, act = case["kind"], case["groups"], case["act"]
    n, c, h, w = st["x"].shape
    dt = st["x"].dtype
    x = st["x"].detach().permute(0, 2, 3, 1).float()
    if kind == "store8":
        return _through_8_bits(x.reshape(-1)).view(n, h, w, c).permute(0, 3, 1, 2).to(dt)
    gamma = st["weight"].detach().float().view(1, 1, groups, c // groups)
    beta = st["bias"].detach().float().view(1, 1, groups, c // groups)
    x = x.reshape(n, h * w, groups, c // groups)
    mean = x.mean((1, 3), keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean((1, 3), keepdim=True) + EPS)
    y = _act(d * rstd * gamma + beta, act).view(n, h, w, c)
    if kind == "packed":
        return y.view(n, h, w, c // 4, 4).permute(0, 3, 1, 2, 4).contiguous().to(dt)
    y = y.permute(0, 3, 1, 2).to(dt)
    if kind == "infer":
        return y
    if kind == "train8":
        x = _through_8_bits(x.reshape(-1)).view_as(x)
        d = x - mean
    xhat = d * rstd
    dy = st["dy"].permute(0, 2, 3, 1).float().reshape(n, h * w, groups, c // groups)
    dz = dy * _act_slope(xhat * gamma + beta, act)
    dweight = (dz * xhat).sum((0, 1)).view(c)
    dbias = dz.sum((0, 1)).view(c)
    dz = dz * gamma
    dx = rstd * (dz - dz.mean((1, 3), keepdim=True) - xhat * (dz * xhat).mean((1, 3), keepdim=True))
    return {"y": y, "dx": dx.view(n, h, w, c).permute(0, 3, 1, 2).to(dt), "dweight": dweight, "dbias": dbias}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ bytes and operations
def work(case):
    b = _BYTES[case["dtype"]]
    e = case["n"] * case["c"] * case["h"] * case["w"]
    eight = e + -(-e // BLOCK)  # a checkpoint: one byte a value and one a block
    c = case["c"]
    kind = case["kind"]
    if kind in ("infer", "packed"):  # x in, y out
        return {"bytes": 2 * b * e + 8 * c, "flops": 12 * e}
    if kind == "store8":  # x in, the checkpoint out and in, the values out
        return {"bytes": 2 * b * e + 2 * eight, "flops": 5 * e}
    if kind == "train":  # forward: x in, y out; backward: dy and x in, dx out
        return {"bytes": 5 * b * e + 24 * c, "flops": 36 * e}
    # forward: x in, y and the checkpoint out; backward: dy and the checkpoint in, dx out
    return {"bytes": 4 * b * e + 2 * eight + 24 * c, "flops": 41 * e}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_8_bits(v):
    """`v` (64 bits, flat) to the multiple of its block's step: 2^(floor(log2 max) - 6), at least
    2^-126, at most 127 steps."""
    full = torch.zeros(-(-v.numel() // BLOCK) * BLOCK, dtype=torch.float64, device=v.device)
    full[:v.numel()] = v
    full = full.view(-1, BLOCK)
    top = full.abs().max(dim=1).values
    _, e = torch.frexp(top)  # top = m 2^e, 1/2 <= m < 1: floor(log2 top) = e - 1
    e = torch.where(top > 0, e - 1, torch.full_like(e, -1000))
    e = (torch.clamp(e, min=-120) - 6).long()[:, None]
    # 2^e and 2^-e from their bits: a power function is an ulp off here and there
    step, per_step = ((1023 + e) << 52).view(torch.float64), ((1023 - e) << 52).view(torch.float64)
    return (torch.clamp((full * per_step).round(), -127.0, 127.0) * step).view(-1)[:v.numel()]


def exact(case, seed):
    st = prepare(case, seed)
    kind, groups, act = case["kind"], case["groups"], case["act"]
    x = st["x"].detach().double()
    n, c, h, w = x.shape

    def eight(v):
        flat = v.permute(0, 2, 3, 1).reshape(-1)
        return _exact_8_bits(flat).view(n, h, w, c).permute(0, 3, 1, 2)

    if kind == "store8":
        return eight(x)
    per_channel = (1, c, 1, 1)
    gamma = st["weight"].detach().double().view(per_channel)
    beta = st["bias"].detach().double().view(per_channel)
    fn = {"elu": torch.nn.functional.elu, "silu": torch.nn.functional.silu, "relu": torch.relu,
          "none": lambda z: z}[act]

    def spread(s):  # [n, groups] to every element
        return s.view(n, groups, 1).expand(n, groups, c // groups).reshape(n, c, 1, 1)

    var, mean = torch.var_mean(x.reshape(n, groups, -1), dim=2, correction=0)
    mean, rstd = spread(mean), spread((var + EPS).rsqrt())
    y = fn((x - mean) * rstd * gamma + beta)
    if kind == "infer":
        return y
    if kind == "packed":
        return y.view(n, c // 4, 4, h, w).permute(0, 1, 3, 4, 2).contiguous()
    if kind == "train8":
        x = eight(x)
    xhat = (x - mean) * rstd
    z = (xhat * gamma + beta).requires_grad_(True)
    dz, = torch.autograd.grad(fn(z), z, st["dy"].double())
    dweight, dbias = (dz * xhat).sum((0, 2, 3)), dz.sum((0, 2, 3))
    u = dz * gamma

    def group_mean(v):
        return spread(v.reshape(n, groups, -1).mean(2))

    dx = rstd * (u - group_mean(u) - xhat * group_mean(u * xhat))
    return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
