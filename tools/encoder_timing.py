"""Time the drop-in's feature encoder (FeaturePyramid, ConvRGBD2, C = 32, laplacian
sigma head) on the GPU at the bench's shape -- both frames of B = 8 pairs, 640x480 --
eager and in the variants `models.LeastSquareTracking` may choose between, and print the
per-kernel breakdown of the NCHW and channels_last calls.

python tools/encoder_timing.py [--batch 16] [--reps 20]
python tools/encoder_timing.py --norm group   # group normalisation: the fused blocks beside the modules in turn
"""
import argparse
import copy
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT]
from deep_prob_feature_track_amd.models.algorithms import FeaturePyramid  # noqa: E402

ap = argparse.ArgumentParser()
ap.add_argument("--batch", type=int, default=16, help="frames (2 per pair)")
ap.add_argument("--reps", type=int, default=20)
ap.add_argument("--down", type=int, default=1)
ap.add_argument("--channels", type=int, default=32)
ap.add_argument("--norm", choices=("batch", "group"), default="batch")
a = ap.parse_args()
dev = torch.device("cuda:0")
torch.manual_seed(0)
enc = FeaturePyramid(D=8, w_uncertainty="laplacian", feature_channel=a.channels, feature_extract="conv",
                     uncertainty_channel=1, norm=a.norm).to(dev).eval()
H, W = 480 // a.down, 640 // a.down
x = torch.randn(a.batch, 8, H, W, device=dev)


def timed(fn, inp):
    with torch.no_grad():
        for _ in range(3):
            fn(inp)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(a.reps):
            fn(inp)
        torch.cuda.synchronize()
    return (time.perf_counter() - t0) / a.reps * 1e3


def max_rel(ref, out):
    worst = 0.0
    for r, o in zip(ref[0] + ref[1], out[0] + out[1]):
        worst = max(worst, ((r - o).abs().max() / r.abs().max().clamp_min(1e-30)).item())
    return worst


with torch.no_grad():
    ref = enc(x)
base = timed(enc, x)
print(f"encoder B={a.batch} {W}x{H} C={a.channels} norm={a.norm}: eager {base:.2f} ms", flush=True)
if a.norm == "group":
    from deep_prob_feature_track_amd.models import submodules
    cl = copy.deepcopy(enc).to(memory_format=torch.channels_last)
    xc = x.contiguous(memory_format=torch.channels_last)
    fused = submodules.ConvBlock._group
    for name, rule, kw in (("fused", fused, {}), ("fused, heads in the solver's layout", fused, dict(packed=True)),
                           ("the modules in turn", lambda self, x: False, {})):
        submodules.ConvBlock._group = rule
        with torch.no_grad():
            out = cl(xc, **kw)
        rel = "" if kw else f", max rel diff {max_rel(ref, out):.2e}"
        print(f"  channels_last, {name}: {timed(lambda t: cl(t, **kw), xc):.2f} ms{rel}", flush=True)
    sys.exit()

def fold_bn(mod):
    """conv -> batchnorm (eval) folded into one conv with bias (rounding differs)."""
    from torch.nn.utils.fusion import fuse_conv_bn_eval
    for m in mod.modules():
        if isinstance(m, torch.nn.Sequential) and len(m) >= 2 and isinstance(m[0], torch.nn.Conv2d) \
                and isinstance(m[1], torch.nn.BatchNorm2d):
            m[0] = fuse_conv_bn_eval(m[0], m[1])
            m[1] = torch.nn.Identity()
    return mod


variants = {"folded BN": (fold_bn(copy.deepcopy(enc)), x)}
cl = copy.deepcopy(enc).to(memory_format=torch.channels_last)
variants["channels_last"] = (cl, x.contiguous(memory_format=torch.channels_last))
variants["folded BN, channels_last"] = (fold_bn(copy.deepcopy(cl)), x.contiguous(memory_format=torch.channels_last))
for name, (mod, inp) in variants.items():
    with torch.no_grad():
        out = mod(inp)
    print(f"  {name}: {timed(mod, inp):.2f} ms, max rel diff {max_rel(ref, out):.2e}", flush=True)
torch.backends.cudnn.benchmark = True
print(f"  eager + MIOpen search: {timed(enc, x):.2f} ms", flush=True)
for name, (mod, inp) in variants.items():
    print(f"  {name} + MIOpen search: {timed(mod, inp):.2f} ms", flush=True)
torch.backends.cudnn.benchmark = False

from torch.profiler import ProfilerActivity, profile  # noqa: E402
for name, mod, inp in (("eager (NCHW)", enc, x), ("channels_last", cl, variants["channels_last"][1])):
    with torch.no_grad(), profile(activities=[ProfilerActivity.CUDA]) as prof:
        for _ in range(3):
            mod(inp)
        torch.cuda.synchronize()
    print(f"--- {name}: 3 calls", flush=True)
    print(prof.key_averages().table(sort_by="cuda_time_total", row_limit=30), flush=True)
