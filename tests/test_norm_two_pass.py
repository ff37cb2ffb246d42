"""The two-pass normalisation kernels where a workgroup visits several blocks of a sample: on the CPU (the kernels in
coroutines, cpu_kernels/norm_values.cpp) and on a MI355X (`-m gpu`) against 64 bits; and the edge cases of fp32 maps
at sizes that the one-launch kernel does not take."""
import math
import os
import re
import subprocess

import pytest
import torch

import norm_oracle as O
from deep_prob_feature_track_amd import _native as N
from deep_prob_feature_track_amd import build as B
from deep_prob_feature_track_amd import norm

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = os.path.join(B.LLVM_BIN, "clang++")
PASSES = ("statistics", "apply", "apply into channel quads", "gradients' sums", "input gradient")

# N, C, H, W, groups.  On the device, with the kernels' own numbers of workgroups: more samples than workgroups, so
# that each walks a sample by itself
DEVICE = [(642, 30, 31, 33, 5),    # a cut row at the end
          (642, 32, 40, 64, 8),    # whole blocks only
          (642, 258, 5, 7, 129),   # statistics and gradients joined by launches of their own
          (642, 7, 41, 61, 1),     # samples of an odd length: a checkpoint's blocks lie anywhere
          (321, 1030, 2, 20, 5)]   # rows of several tiles
WIDE = (330, 512, 12, 12, 1)       # channel quads in tiles of their own
# on the CPU, with few workgroups: 1 or 2 samples, 2 to 6 workgroups each
FEW = {"kStatsWorkgroups": 4, "kSumsWorkgroups": 4, "kApplyWorkgroups": 6, "kGradWorkgroups": 6}
SMALL = [(2, 30, 31, 43, 5), (2, 32, 40, 64, 8), (2, 258, 9, 17, 129), (2, 7, 79, 83, 1), (2, 1030, 5, 8, 5),
         (2, 4, 131, 101, 1), (2, 6, 110, 77, 3), (1, 16, 80, 72, 8), (1, 36, 63, 64, 3), (1, 512, 12, 13, 1)]
EDGES = [(2, 30, 30, 40, 5), (1, 32, 64, 80, 8)]  # (D % 4 != 0; more pixels than a workgroup holds)


def _map(n, c, h, w, dtype, seed=0, offset=0.0, dev="cpu"):
    """A convolution's output: channels of unlike mean and spread, channels_last."""
    g = torch.Generator().manual_seed(5000 + seed)
    x = torch.randn(n, h, w, c, generator=g) * torch.exp(0.5 * torch.randn(c, generator=g)) \
        + torch.randn(c, generator=g) + offset
    return x.to(dtype).to(dev).permute(0, 3, 1, 2)


def _params(c, seed=0, dev="cpu"):
    g = torch.Generator().manual_seed(6000 + seed)
    return (1 + 0.3 * torch.randn(c, generator=g)).to(dev), (0.3 * torch.randn(c, generator=g)).to(dev)


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


# ------------------------------------------------------------------ on the CPU
@pytest.fixture(scope="module")
def binary(tmp_path_factory):
    """norm_values over the kernels' source, whose numbers of workgroups its command line may change."""
    if not os.path.exists(CLANG):
        pytest.skip("no clang++ that knows vector types and 16-bit floats")
    source = open(os.path.join(B.CSRC, "dpft_norm.hip")).read()
    names = ", ".join(rf"{name} = \d+" for name in FEW)
    source, count = re.subn(rf"constexpr int ({names});", r"static int \1;", source)
    assert count == 1
    folder = tmp_path_factory.mktemp("norm_values")
    (folder / "dpft_norm.hip").write_text(source)
    bounds = open(os.path.join(HERE, "cpu_kernels", "norm_bounds.cpp")).read()
    include = '#include "../../deep_prob_feature_track_amd/csrc/dpft_norm.hip"'
    assert bounds.count(include) == 1
    (folder / "norm_bounds.cpp").write_text(bounds.replace(include, '#include "dpft_norm.hip"'))
    (folder / "norm_values.cpp").write_text(open(os.path.join(HERE, "cpu_kernels", "norm_values.cpp")).read())
    out = str(folder / "norm_values")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O0", "-w", f"-I{HERE}/cpu_kernels", f"-I{B.INC}", f"-I{B.CSRC}",
                    str(folder / "norm_values.cpp"), "-o", out], check=True)
    return out


def _walk(binary, shape, dtype, few=()):
    """(blocks, workgroups) of a sample's tile for each pass, tiles, whether the one-launch kernel takes it."""
    r = subprocess.run([binary, "walk", *map(str, shape), str(N.TYPES[dtype]), *map(str, few)], capture_output=True,
                       text=True, check=True)
    v = [int(t) for t in r.stdout.split()]
    return list(zip(v[0:10:2], v[1:10:2])), v[10], bool(v[11])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", DEVICE + [WIDE])
def test_device_sizes_loop(binary, shape, dtype):
    """The sizes of the device tests give a workgroup several blocks in every pass."""
    if shape == WIDE and dtype != F32:
        pytest.skip("channel quads are fp32")
    walks, _, one_launch = _walk(binary, shape, dtype)
    assert not one_launch
    for what, (blocks, parts) in zip(PASSES, walks):
        assert blocks > parts or (shape == WIDE) != (what == PASSES[2]), (what, blocks, parts)


@pytest.mark.parametrize("shape", EDGES)
def test_edge_sizes_take_two_passes(binary, shape):
    """... and those of the edge cases several records a sample, in fp32."""
    walks, _, one_launch = _walk(binary, shape, F32)
    assert not one_launch and walks[0][1] > 1 and walks[3][1] > 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SMALL)
def test_values_on_the_cpu(binary, shape, dtype):
    """y, the checkpoint, the channel quads and both backward passes of each size."""
    n, c, h, w, groups = shape
    walks, _, one_launch = _walk(binary, shape, dtype, FEW.values())
    assert not one_launch
    for k, (what, (blocks, parts)) in enumerate(zip(PASSES, walks)):
        assert k == 2 or blocks > parts, (what, blocks, parts)
    # a thread's terms in a row: 8 or 4 vectors a block; 64 more for the joins over its neighbours (norm_oracle)
    run = 64 + max(math.ceil(walks[0][0] / walks[0][1]) * 8, math.ceil(walks[3][0] / walks[3][1]) * 4)
    total, size = n * c * h * w, 2 if dtype != F32 else 4
    i = (SMALL.index(shape) + TYPES.index(dtype)) % 2
    for name in (("elu", "silu")[i],):
        x, dy = _map(n, c, h, w, dtype, seed=i), _map(n, c, h, w, dtype, seed=50 + i)
        wt, b = _params(c, i)

        def raw(t):
            return t.contiguous().view(torch.uint8).numpy().tobytes()
        data = raw(x.permute(0, 2, 3, 1)) + raw(dy.permute(0, 2, 3, 1)) + raw(wt) + raw(b)
        r = subprocess.run([binary, "run", *map(str, shape), str(N.TYPES[dtype]), *map(str, FEW.values()),
                            str(N.ACTS[name])], input=data, capture_output=True, timeout=600)
        assert r.returncode == 0, r.stderr.decode()
        out, at = bytearray(r.stdout), 0

        def take(count, t, each):
            nonlocal at
            v = torch.frombuffer(out, dtype=t, count=count, offset=at)
            at += count * each
            return v

        def whole():
            return take(total, dtype, size).view(n, h, w, c).permute(0, 3, 1, 2)
        y, q, scale = whole(), take(total, torch.int8, 1), take(-(-total // 32), torch.uint8, 1)
        want, codes = O.through_8_bits(x.permute(0, 2, 3, 1).reshape(-1).double())
        step = ((codes + (1023 - 133)) << 52).view(torch.float64).repeat_interleave(32)[:total]
        assert torch.equal(scale.long(), codes) and torch.equal(q.double() * step, want)
        if dtype == F32 and c % 4 == 0:
            packed = take(total, dtype, size).view(n, c // 4, h, w, 4)
            assert torch.equal(packed.permute(0, 1, 4, 2, 3).reshape(n, c, h, w), y)
        for checkpoint in (False, True):
            ref = O.Reference(x, groups, wt, b, 1e-5, name, dy, checkpoint=checkpoint, run=run)
            dx, dw, db = whole(), take(c, F32, 4), take(c, F32, 4)
            for what, got, exact, tol in (("y", y, ref.y, ref.y_tol), ("dx", dx, ref.dx, ref.dx_tol),
                                          ("dweight", dw, ref.dweight, 1.01 * ref.dweight_tol + O.U * ref.dweight.abs()),
                                          ("dbias", db, ref.dbias, 1.01 * ref.dbias_tol + O.U * ref.dbias.abs())):
                assert O.excess(got, exact, tol) <= 0, (what, name, checkpoint)
        assert at == len(out)


# ------------------------------------------------------------------ on the device
def _run(shape, dtype):
    """Terms in a row where a workgroup walks a sample by itself: at least 65 of its threads' vectors side by side."""
    n, c, h, w, _ = shape
    return 64 + math.ceil(h * w * c / (64 * (4 if dtype == F32 else 8)))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", DEVICE)
def test_forward_and_backward(shape, dtype):
    dev = _dev()
    n, c, h, w, groups = shape
    x = _map(n, c, h, w, dtype, seed=1, dev=dev).requires_grad_(True)
    wt, b = (p.requires_grad_(True) for p in _params(c, 1, dev=dev))
    dy = _map(n, c, h, w, dtype, seed=51, dev=dev)
    for ck in (False, True):
        y = norm.group_norm_act(x, groups, wt, b, checkpoint=ck)
        dx, dw, db = torch.autograd.grad(y, (x, wt, b), dy)
        r = O.Reference(x, groups, wt, b, 1e-5, "elu", dy, checkpoint=ck, run=_run(shape, dtype))
        assert O.excess(y, r.y, r.y_tol) <= 0 and O.excess(dx, r.dx, r.dx_tol) <= 0
        assert O.excess(dw, r.dweight, 1.01 * r.dweight_tol + O.U * r.dweight.abs()) <= 0
        assert O.excess(db, r.dbias, 1.01 * r.dbias_tol + O.U * r.dbias.abs()) <= 0
        with torch.no_grad():
            assert torch.equal(norm.group_norm_act(x, groups, wt, b), y)
        del r, y, dx, dw, db


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", DEVICE)
def test_every_value_counts_once(shape, dtype):
    """Gradients of whole numbers through no activation: their sums are exact in fp32, so that one value left out
    or read twice shows, wherever it lies.  (At most 2 x 642 x 2560 < 2^24.)"""
    dev = _dev()
    n, c, h, w, groups = shape
    x = _map(n, c, h, w, dtype, seed=2, dev=dev)
    dy = torch.randint(-2, 3, (n, h, w, c), generator=torch.Generator().manual_seed(7)).to(dtype).to(dev).permute(0, 3, 1, 2)
    want = dy.double().sum((0, 2, 3))
    for ck in (False, True):
        b = torch.zeros(c, device=dev, requires_grad=True)
        y = norm.group_norm_act(x, groups, None, b, act="none", checkpoint=ck)
        assert torch.equal(torch.autograd.grad(y, b, dy)[0].double(), want)


@gpu
@pytest.mark.parametrize("shape", [DEVICE[1], WIDE])
def test_channel_quads(shape):
    from deep_prob_feature_track_amd import ic
    dev = _dev()
    n, c, h, w, groups = shape
    x, (wt, b) = _map(n, c, h, w, F32, seed=3, dev=dev), _params(c, 3, dev=dev)
    y = norm.group_norm_act(x, groups, wt, b)
    assert torch.equal(norm.group_norm_act(x, groups, wt, b, packed=True), ic.pack_features(y.contiguous()))
    r = O.Reference(x, groups, wt, b, 1e-5, "elu", run=_run(shape, F32))
    assert O.excess(y, r.y, r.y_tol) <= 0


# ------------------------------------------------------------------ edge cases in fp32
@gpu
@pytest.mark.parametrize("shape", EDGES)
@pytest.mark.parametrize("offset", [1e3, 1e4, -1e4])
def test_far_mean(shape, offset):
    """The statistics of values far from 0: taken from squares, 0.06 or 6 times the spread's square would be lost
    (offset^2 U).  The bounds of norm_oracle with a mean that is off by 32 U of itself: a mean of 8 values in a row by
    4.4 U, at most 9 joins over neighbours and 6 over lanes by U each.  A part's mean that is off by e changes the
    squares about the whole's by 2 e |mean - part's mean| + e^2, of which the first comes to at most 2 e times the
    spread: rstd is off by e rstd + (e rstd)^2 of itself."""
    dev = _dev()
    n, c, h, w, groups = shape
    x = _map(n, c, h, w, F32, seed=4, offset=offset, dev=dev).requires_grad_(True)
    wt, b = (p.requires_grad_(True) for p in _params(c, 4, dev=dev))
    dy = _map(n, c, h, w, F32, seed=54, dev=dev)
    y = norm.group_norm_act(x, groups, wt, b, act="silu")
    dx, dw, db = torch.autograd.grad(y, (x, wt, b), dy)
    r = O.Reference(x, groups, wt, b, 1e-5, "silu", dy)
    far = 32 * O.U * abs(offset) * 1.01  # the mean's own error
    rstd = r.rstd.repeat_interleave(c // groups, 1).view(n, c, 1, 1)
    xhat = (x.detach().double() - r.mean.repeat_interleave(c // groups, 1).view(n, c, 1, 1)) * rstd
    g = wt.detach().double().view(1, c, 1, 1).abs()
    rstd_off = far * rstd + (far * rstd) ** 2  # of itself
    off = far * rstd * (1 + rstd_off) + xhat.abs() * rstd_off  # of xhat
    assert off.max() < 0.2  # (far below what a lost spread would do)
    assert O.excess(y, r.y, r.y_tol + 1.1 * g * off) <= 0
    # the slope's derivative is at most 1/2 for silu, the slope at most 1.1
    d = dy.double().abs()
    u_off = d * 0.5 * g * off
    assert O.excess(db, r.dbias, 1.01 * r.dbias_tol + u_off.sum((0, 2, 3))) <= 0
    w_off = u_off * (xhat.abs() + off) + 1.1 * d * off
    assert O.excess(dw, r.dweight, 1.01 * r.dweight_tol + w_off.sum((0, 2, 3))) <= 0

    def gmean(v):
        return v.reshape(n, groups, -1).mean(2).repeat_interleave(c // groups, 1).view(n, c, 1, 1)
    m2 = gmean(1.1 * d * g * (xhat.abs() + off))
    dx_off = rstd * (g * u_off + gmean(g * u_off) + (xhat.abs() + off) * gmean(g * w_off) + off * m2)
    dx_off = dx_off * (1 + rstd_off) + rstd_off * rstd * (1.1 * d * g + gmean(1.1 * d * g) + (xhat.abs() + off) * m2)
    assert O.excess(dx, r.dx, r.dx_tol + dx_off) <= 0


@gpu
@pytest.mark.parametrize("shape", EDGES)
def test_an_outlier(shape):
    dev = _dev()
    n, c, h, w, groups = shape
    for at in ((0, 0), (h // 2, w // 3), (h - 1, w - 1)):
        x = _map(n, c, h, w, F32, seed=5, dev=dev).clone(memory_format=torch.channels_last)
        x[:, :, at[0], at[1]] = 1e4
        y = norm.group_norm_act(x, groups, act="none")
        r = O.Reference(x, groups, None, None, 1e-5, "none")
        assert O.excess(y, r.y, r.y_tol) <= 0


@gpu
@pytest.mark.parametrize("shape", EDGES)
def test_non_finite_values_stay_in_their_group(shape):
    """... of their sample, forward and backward: y, dx, and the gradients of the group's own channels."""
    dev = _dev()
    n, c, h, w, groups = shape
    d = c // groups
    x = _map(n, c, h, w, F32, seed=6, dev=dev)
    wt, b = (p.requires_grad_(True) for p in _params(c, 6, dev=dev))
    dy = _map(n, c, h, w, F32, seed=56, dev=dev)

    def step(x, ck):
        x = x.detach().requires_grad_(True)
        y = norm.group_norm_act(x, groups, wt, b, checkpoint=ck)
        return (y.detach(),) + torch.autograd.grad(y, (x, wt, b), dy)
    keep = torch.ones(n, c, h, w, dtype=torch.bool, device=dev)
    keep[n - 1, d:2 * d] = False  # group 1 of the last sample
    for ck in (False, True):
        ref = step(x, ck)
        for bad in (float("nan"), float("inf"), -float("inf")):
            for px in ((3, 4), (h - 1, w - 1)):
                z = x.clone(memory_format=torch.channels_last)
                z[n - 1, 2 * d - 1, px[0], px[1]] = bad
                y, dx, dw, db = step(z, ck)
                assert y[~keep].isnan().all() and torch.equal(y[keep], ref[0][keep])
                assert dx[~keep].isnan().all()
                assert dw[d:2 * d].isnan().all()
                others = torch.ones(c, dtype=torch.bool, device=dev)
                others[d:2 * d] = False
                if not ck:  # (a checkpoint's block of 32 values, NaN as a whole, reaches into other groups' gradients)
                    assert torch.equal(dx[keep], ref[1][keep])
                    assert torch.equal(dw[others], ref[2][others]) and torch.equal(db[others], ref[3][others])


@gpu
@pytest.mark.parametrize("shape", EDGES)
def test_constant_group(shape):
    """No spread: xhat = 0, y = act(bias), and a gradient that its own mean and xhat = 0 leave."""
    dev = _dev()
    n, c, h, w, groups = shape
    x = torch.full((n, c, h, w), 3.25, device=dev).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    wt, b = (p.requires_grad_(True) for p in _params(c, 7, dev=dev))
    dy = _map(n, c, h, w, F32, seed=57, dev=dev)
    y = norm.group_norm_act(x, groups, wt, b)
    r = O.Reference(x, groups, wt, b, 1e-5, "elu", dy)
    assert O.excess(y, r.y, r.y_tol) <= 0
    dx, dw, db = torch.autograd.grad(y, (x, wt, b), dy)
    assert O.excess(dx, r.dx, r.dx_tol) <= 0 and O.excess(dw, r.dweight, r.dweight_tol * 1.01 + 1e-30) <= 0
    assert O.excess(db, r.dbias, r.dbias_tol * 1.01) <= 0


@gpu
@pytest.mark.parametrize("shape", EDGES)
def test_relu(shape):
    """relu's slope jumps at 0: dy is 0 where z is within its own error of it."""
    dev = _dev()
    n, c, h, w, groups = shape
    x = _map(n, c, h, w, F32, seed=8, dev=dev).requires_grad_(True)
    wt, b = (p.requires_grad_(True) for p in _params(c, 8, dev=dev))
    r = O.Reference(x, groups, wt, b, 1e-5, "relu")
    dy = _map(n, c, h, w, F32, seed=58, dev=dev) * (r.z.abs() > 4 * r.z_tol)
    y = norm.group_norm_act(x, groups, wt, b, act="relu")
    r = O.Reference(x, groups, wt, b, 1e-5, "relu", dy)
    dx, dw, db = torch.autograd.grad(y, (x, wt, b), dy)
    assert O.excess(y, r.y, r.y_tol) <= 0 and O.excess(dx, r.dx, r.dx_tol) <= 0
    assert O.excess(dw, r.dweight, r.dweight_tol * 1.01) <= 0 and O.excess(db, r.dbias, r.dbias_tol * 1.01) <= 0
