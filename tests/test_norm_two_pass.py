"""The two-pass normalisation kernels where a workgroup visits several blocks of a sample: on the CPU (the kernels in
coroutines, cpu_kernels/norm_values.cpp) and on a MI355X (`-m gpu`) against 64 bits."""
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
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-w", f"-I{HERE}/cpu_kernels", f"-I{B.INC}", f"-I{B.CSRC}",
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
