"""The package's modules import, and their torch paths run, where the built libraries cannot be loaded (stale, half
written, of another torch, missing): only the calls that need them raise."""
import os
import shutil
import subprocess
import sys

import pytest

import deep_prob_feature_track_amd as pkg

HERE = os.path.dirname(os.path.abspath(pkg.__file__))
LIBS = ("libdpft_ic.so", "libdpft_torch.so")
SCRIPT = """
import torch
from deep_prob_feature_track_amd.models import LeastSquareTracking, submodules
from deep_prob_feature_track_amd import norm
x = torch.randn(1, 4, 8, 8)
for kind in ("batch", "group"):
    assert submodules.convLayer(True, 4, 8, norm=kind)(x).shape == (1, 8, 8, 8)
for call in (lambda: norm.group_norm_act(x, 2), lambda: norm.act_checkpoint(x)):
    for again in range(2):
        try:
            call()
        except (OSError, RuntimeError, AttributeError) as e:
            assert "libdpft" in str(e), e
        else:
            raise SystemExit("no error")
print("ran")
"""


@pytest.mark.parametrize("broken,how", [(LIBS, "cut"), (LIBS[1:], "cut"), (LIBS[:1], "cut"), (LIBS, "empty"),
                                        (LIBS, "missing")], ids=["both", "torch", "solver", "empty", "missing"])
def test_import_and_torch_paths(broken, how, tmp_path):
    for lib in LIBS:
        if not os.path.exists(os.path.join(HERE, lib)):
            pytest.skip(f"{lib} is not built")
    copy = tmp_path / "deep_prob_feature_track_amd"
    shutil.copytree(HERE, copy, ignore=shutil.ignore_patterns("csrc", "data", "__pycache__", "*.o", "*.json"))
    for lib in broken:
        data = (copy / lib).read_bytes()
        (copy / lib).unlink()
        if how != "missing":
            (copy / lib).write_bytes(data[:len(data) // 2] if how == "cut" else b"")
    env = dict(os.environ, PYTHONPATH=str(tmp_path))
    r = subprocess.run([sys.executable, "-c", SCRIPT], cwd=tmp_path, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ran\n", r.stderr
