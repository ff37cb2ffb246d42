"""A group-norm block's result under autocast has the convolution's type in every layout and with hooks, as a
batch-norm block's has."""
import pytest
import torch
import torch.nn.functional as F

import norm_oracle as O
from deep_prob_feature_track_amd.models import submodules
from deep_prob_feature_track_amd.models.submodules import convLayer

gpu = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


def _block():
    torch.manual_seed(3)
    blk = convLayer(True, 8, 24, 1, norm="group")
    with torch.no_grad():
        blk[1].weight.add_(0.3 * torch.randn(24))
        blk[1].bias.add_(0.3 * torch.randn(24))
    return blk


@pytest.mark.parametrize("dtype", HALVES)
def test_modules_in_turn_return_the_maps_type(dtype, monkeypatch):
    """Autocast's policy for group norm on a device (its inputs in fp32, the result too) put in its place."""
    plain = F.group_norm
    monkeypatch.setattr(F, "group_norm", lambda x, n, w, b, eps: plain(x.float(), n, w, b, eps))
    monkeypatch.setattr(submodules.gn, "group_norm_act", lambda *a, **k: pytest.fail("the modules should run"))
    blk, y = _block(), torch.randn(2, 24, 5, 7).to(dtype)
    want = F.elu(plain(y.float(), 8, blk[1].weight, blk[1].bias)).to(dtype)
    got = blk._group_epilogue(y)
    assert got.dtype == dtype and torch.equal(got, want)  # rounded once, at the end


@gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_every_layout_returns_the_maps_type(dtype):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    dev = torch.device("cuda:0")
    blk = _block().to(dev)
    nchw = torch.randn(2, 24, 9, 11, generator=torch.Generator().manual_seed(4)).to(dtype).to(dev)
    # 297 values to a group: the modules' statistics are sums of them in fp32, in an order of the library's own
    r = O.Reference(nchw, 8, blk[1].weight, blk[1].bias, blk[1].eps, "elu", run=300)
    hooked = _block().to(dev)
    hooked[1].register_forward_hook(lambda m, i, o: None)
    nhwc = nchw.contiguous(memory_format=torch.channels_last)
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        for b, y in ((blk, nhwc), (blk, nchw), (blk, nchw[:, :, :, 1:]), (hooked, nhwc), (hooked, nchw)):
            got = b._group_epilogue(y)
            assert got.dtype == dtype
            if y.shape == nchw.shape:
                assert O.excess(got, r.y, r.y_tol) <= 0
    for b, y in ((blk, nhwc), (blk, nchw)):  # in training too: a leaf's gradient has its type
        y = y.clone(memory_format=torch.preserve_format).requires_grad_(True)
        with torch.autocast("cuda", dtype=dtype):
            out = b._group_epilogue(y)
        assert out.dtype == dtype
        assert torch.autograd.grad(out, y, torch.ones_like(out))[0].dtype == dtype
