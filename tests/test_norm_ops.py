"""Group normalisation with an activation and 8-bit activation checkpoints: refusals and the format on
the CPU, the kernels against their 64-bit definitions (tests/norm_oracle.py) on a MI355X (`-m gpu`)."""
import ctypes

import pytest
import torch

import norm_oracle as O
from deep_prob_feature_track_amd import _native as N
from deep_prob_feature_track_amd import norm

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


def _map(n, c, h, w, dtype, seed=0, offset=0.0, dev="cpu"):
    """A convolution's output: channels of unlike mean and spread, channels_last."""
    g = torch.Generator().manual_seed(1000 + seed)
    x = torch.randn(n, h, w, c, generator=g) * torch.exp(0.5 * torch.randn(c, generator=g)) \
        + torch.randn(c, generator=g) + offset
    return x.to(dtype).to(dev).permute(0, 3, 1, 2)


def _params(c, seed=0, dtype=F32, dev="cpu"):
    g = torch.Generator().manual_seed(2000 + seed)
    return ((1 + 0.3 * torch.randn(c, generator=g)).to(dtype).to(dev),
            (0.3 * torch.randn(c, generator=g)).to(dtype).to(dev))


# ------------------------------------------------------------------ without a GPU
def test_oracle_gradients_match_differences():
    """The oracle's dx, dweight and dbias against central differences of its own y in 64 bits."""
    for name in ("none", "elu", "silu"):
        x = _map(2, 6, 4, 5, F32).double()
        w, b = (p.double() for p in _params(6))
        dy = torch.randn(2, 6, 4, 5, generator=torch.Generator().manual_seed(5)).double()
        r = O.Reference(x, 3, w, b, 1e-5, name, dy)
        for t, grad in ((x, r.dx), (w, r.dweight), (b, r.dbias)):
            v = torch.randn(t.shape, generator=torch.Generator().manual_seed(6)).double()
            h = 1e-5
            ys = []
            for s in (h, -h):
                a = [u + s * v if u is t else u for u in (x, w, b)]
                ys.append((O.Reference(a[0], 3, a[1], a[2], 1e-5, name).y * dy).sum())
            assert abs((ys[0] - ys[1]) / (2 * h) - (grad * v).sum()) < 1e-7


def test_refusals():
    x = torch.zeros(2, 6, 4, 4)
    ones = torch.ones(6)
    for kw, err in ((dict(groups=4), ValueError), (dict(groups=0), ValueError), (dict(groups=3, act="tanh"), ValueError),
                    (dict(groups=3, eps=-1.0), ValueError), (dict(groups=3, eps=float("nan")), ValueError),
                    (dict(groups=3, weight=torch.ones(5)), ValueError),
                    (dict(groups=3, bias=torch.ones(6, dtype=torch.float64)), TypeError),
                    (dict(groups=3, weight=ones, bias=ones.half()), TypeError),
                    (dict(groups=3, packed=True), ValueError),  # C % 4
                    (dict(groups=3, weight=ones.clone().requires_grad_(True), packed=True), RuntimeError),
                    (dict(groups=3), RuntimeError)):  # a CPU tensor
        with pytest.raises(err):
            norm.group_norm_act(x, **kw)
    with pytest.raises(ValueError):
        norm.group_norm_act(x[0], 3)
    with pytest.raises(TypeError):
        norm.group_norm_act(x.double(), 3)
    with pytest.raises(RuntimeError):
        norm.act_checkpoint(x)
    with pytest.raises(TypeError):
        norm.act_checkpoint(x.int())
    with pytest.raises(RuntimeError):
        norm.conv2d(x, torch.zeros(2, 6, 1, 1))
    with pytest.raises(ValueError):
        norm.conv2d(x, torch.zeros(2, 6, 1, 1), padding="same")


def test_entry_points_refuse_without_device_work():
    L = N.lib()
    p = ctypes.c_void_p(4096)
    good = dict(pixels=16, N=1, C=8, groups=2, act=2, x_type=0, param_type=0, flags=0, eps=1e-5)

    def desc(**kw):
        return ctypes.byref(N.GroupNorm(*{**good, **kw}.values()))
    assert L.dpft_group_norm_workspace_size(desc()) > 0
    for bad in (dict(pixels=0), dict(N=0), dict(C=0), dict(groups=3), dict(groups=-1), dict(act=4), dict(act=-1),
                dict(x_type=3), dict(param_type=-1), dict(flags=2), dict(eps=-1.0), dict(eps=float("nan")),
                dict(flags=1, x_type=1), dict(flags=1, C=6), dict(pixels=1 << 50), dict(N=1 << 30), dict(C=1 << 28)):
        assert L.dpft_group_norm_workspace_size(desc(**bad)) == 0, bad
        assert L.dpft_group_norm_act(desc(**bad), p, p, p, ctypes.c_void_p(8192), None, None, None, None, p, 1 << 30,
                                     None) == -1
        assert L.dpft_last_error()
    ws = L.dpft_group_norm_workspace_size(desc())
    y = ctypes.c_void_p(1 << 20)

    def fwd(x=p, out=y, q=None, s=None, w=p, nb=ws, **kw):
        return L.dpft_group_norm_act(desc(**kw), x, p, p, out, None, None, q, s, w, nb, None)
    assert fwd(x=None) == fwd(out=None) == fwd(w=None) == fwd(out=p) == fwd(q=p) == fwd(s=p) == -1
    assert fwd(q=p, s=p, flags=1) == -1 and fwd(x=ctypes.c_void_p(4100)) == -1 and fwd(nb=ws - 1) == -2

    def bwd(dy=p, x=p, q=None, s=None, m=p, dx=y, nb=ws, **kw):
        return L.dpft_group_norm_act_backward(desc(**kw), dy, x, q, s, p, p, m, p, dx, p, p, p, nb, None)
    assert bwd(dy=None) == bwd(x=None) == bwd(x=None, q=p) == bwd(q=p, s=p) == bwd(m=None) == bwd(dx=p) == -1
    assert bwd(flags=1) == -1 and bwd(dy=ctypes.c_void_p(4104)) == -1 and bwd(nb=0) == -2
    for f in (lambda t, n, a: L.dpft_act_checkpoint(a, t, n, p, p, None),
              lambda t, n, a: L.dpft_act_restore(a, p, n, y, t, None)):
        assert f(3, 8, p) == f(0, 0, p) == f(0, 8, None) == f(0, 8, ctypes.c_void_p(4097)) == f(0, 1 << 60, p) == -1


@pytest.mark.parametrize("checkpoint", [False, True])
def test_traces_with_symbolic_sizes(checkpoint):
    """Forward and backward in a trace whose batch and pixels are symbols: the operators, shapes and layouts."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(x, w, b):
        y = norm.group_norm_act(x, 4, w, b, checkpoint=checkpoint)
        return (y,) + torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    x = _map(2, 8, 6, 10, F32).requires_grad_(True)
    w, b = (p.requires_grad_(True) for p in _params(8))
    g = make_fx(step, tracing_mode="symbolic", _allow_non_fake_inputs=True)(x, w, b)
    names = [n.target.__name__ for n in g.graph.nodes if n.op == "call_function"]
    assert names.count("group_norm_act_forward.default") == names.count("group_norm_act_backward.default") == 1
    out = [n for n in g.graph.nodes if n.op == "output"][0].args[0]
    y, dx, dw, db = (n.meta["val"] for n in out)
    assert not isinstance(y.shape[2], int)  # a symbol
    assert y.stride(1) == dx.stride(1) == 1 and y.dtype == F32 and dw.shape == db.shape == (8,)
    p = make_fx(lambda t: norm.group_norm_act(t, 4, packed=True), tracing_mode="symbolic")(x.detach())
    assert [n for n in p.graph.nodes if n.op == "output"][0].args[0].meta["val"].dim() == 5


# ------------------------------------------------------------------ the kernels
SHAPES = [  # N, C, H, W, groups
    (1, 1, 1, 1, 1), (2, 6, 1, 1, 3), (1, 8, 5, 7, 2), (3, 30, 9, 11, 5), (2, 13, 17, 5, 1), (1, 7, 3, 50, 7),
    (1, 32, 64, 80, 8), (2, 96, 15, 20, 8), (16, 16, 9, 9, 4), (1, 300, 7, 3, 4), (1, 257, 3, 5, 1),
    (2, 1030, 2, 3, 5), (1, 2056, 1, 3, 8), (5, 64, 33, 1, 64), (1, 4, 300, 301, 1),
    (2, 258, 5, 6, 129), (1, 400, 9, 7, 200)]  # (groups of a launch of their own)


def _check(r, y=None, dx=None, dw=None, db=None, p_half=O.U):
    if y is not None:
        assert O.excess(y, r.y, r.y_tol) <= 0, "y"
    if dx is not None:
        assert O.excess(dx, r.dx, r.dx_tol) <= 0, "dx"
    if dw is not None:
        assert O.excess(dw, r.dweight, r.dweight_tol * 1.01 + p_half * r.dweight.abs()) <= 0, "dweight"
    if db is not None:
        assert O.excess(db, r.dbias, r.dbias_tol * 1.01 + p_half * r.dbias.abs()) <= 0, "dbias"


def _grads(y, ins, dy):
    return torch.autograd.grad(y, ins, dy)


@gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_forward_and_backward(shape, dtype):
    dev = _dev()
    n, c, h, w, groups = shape
    for i, name in enumerate(("elu", "silu", "none")):
        x = _map(n, c, h, w, dtype, seed=i, dev=dev).requires_grad_(True)
        wt, b = (p.requires_grad_(True) for p in _params(c, i, dev=dev))
        dy = _map(n, c, h, w, dtype, seed=50 + i, dev=dev)
        for ck in (False, True):
            y = norm.group_norm_act(x, groups, wt, b, act=name, checkpoint=ck)
            assert y.dtype == dtype and y.is_contiguous(memory_format=torch.channels_last)
            r = O.Reference(x, groups, wt, b, 1e-5, name, dy, checkpoint=ck)
            _check(r, y, *_grads(y, (x, wt, b), dy))
            with torch.no_grad():
                assert torch.equal(norm.group_norm_act(x, groups, wt, b, act=name), y)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_relu(dtype):
    """relu's slope jumps at 0: dy is 0 where z is within its own error of it."""
    dev = _dev()
    x = _map(2, 24, 19, 23, dtype, dev=dev).requires_grad_(True)
    wt, b = (p.requires_grad_(True) for p in _params(24, dev=dev))
    r = O.Reference(x, 6, wt, b, 1e-5, "relu")
    dy = _map(2, 24, 19, 23, dtype, seed=9, dev=dev) * (r.z.abs() > 4 * r.z_tol)
    y = norm.group_norm_act(x, 6, wt, b, act="relu")
    _check(O.Reference(x, 6, wt, b, 1e-5, "relu", dy), y, *_grads(y, (x, wt, b), dy))


@gpu
@pytest.mark.parametrize("c,h,w", [(32, 24, 40), (4, 3, 5), (20, 7, 9), (36, 40, 41), (512, 30, 21)])
def test_packed_layout(c, h, w):
    """The channel-quad output holds the plain output's bits."""
    from deep_prob_feature_track_amd import ic
    dev = _dev()
    x = _map(3, c, h, w, F32, dev=dev)
    wt, b = _params(c, dev=dev)
    y = norm.group_norm_act(x, 4, wt, b)
    p = norm.group_norm_act(x, 4, wt, b, packed=True)
    assert p.shape == (3, c // 4, h, w, 4) and torch.equal(p, ic.pack_features(y.contiguous()))


@gpu
def test_parameters_optional_and_typed():
    dev = _dev()
    x = _map(2, 16, 9, 10, BF16, dev=dev).requires_grad_(True)
    dy = _map(2, 16, 9, 10, BF16, seed=3, dev=dev)
    y = norm.group_norm_act(x, 4)
    _check(O.Reference(x, 4, None, None, 1e-5, "elu", dy), y, *_grads(y, (x,), dy))
    wt, b = (p.requires_grad_(True) for p in _params(16, dtype=BF16, dev=dev))
    for ws, bs, ins in ((wt, b, (x, wt, b)), (wt, None, (wt,)), (None, b, (b,))):
        y = norm.group_norm_act(x, 4, ws, bs)
        r = O.Reference(x, 4, ws, bs, 1e-5, "elu", dy)
        for i, g in zip(ins, _grads(y, ins, dy)):
            assert g.dtype == i.dtype
            kw = {"dx": g} if i is x else {"dw": g} if i is wt else {"db": g}
            _check(r, y, p_half=torch.finfo(BF16).eps / 2 * 1.01, **kw)


@gpu
def test_layouts_and_alignment():
    """NCHW storage, a channel slice of a wider map, an offset view, a broadcast gradient."""
    dev = _dev()
    wt, b = (p.requires_grad_(True) for p in _params(10, dev=dev))
    base = _map(2, 10, 12, 14, F32, dev=dev)
    wide = torch.cat((base, base), 1).contiguous(memory_format=torch.channels_last)
    store = torch.zeros(base.numel() + 1, device=dev)
    store[1:] = base.permute(0, 2, 3, 1).reshape(-1)
    off = store[1:].view(2, 12, 14, 10).permute(0, 3, 1, 2)
    dy = torch.ones(1, 1, 1, 1, device=dev).expand(2, 10, 12, 14)
    r = O.Reference(base, 5, wt, b, 1e-5, "elu", dy)
    for x in (base.contiguous(), wide[:, 10:], off):
        x = x.detach().requires_grad_(True)
        y = norm.group_norm_act(x, 5, wt, b)
        _check(r, y, *_grads(y, (x, wt, b), dy))
    with torch.no_grad():
        assert torch.equal(norm.group_norm_act(base, 5, wt[::1], b), norm.group_norm_act(off, 5, wt, b))


@gpu
def test_empty_maps():
    dev = _dev()
    wt, b = (p.requires_grad_(True) for p in _params(8, dev=dev))
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        for ck in (False, True):
            y = norm.group_norm_act(x, 2, wt, b, checkpoint=ck)
            dx, dw, db = _grads(y, (x, wt, b), torch.zeros_like(y))
            assert y.shape == shape and dx.shape == shape and not dw.any() and not db.any()
        assert norm.act_restore(norm.act_checkpoint(x)).shape == shape


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_far_mean(dtype):
    """A mean far from 0: the spread has to come from differences, not from squares."""
    dev = _dev()
    x = _map(2, 16, 30, 40, dtype, offset=300.0, dev=dev).requires_grad_(True)
    wt, b = (p.requires_grad_(True) for p in _params(16, dev=dev))
    dy = _map(2, 16, 30, 40, dtype, seed=4, dev=dev)
    y = norm.group_norm_act(x, 4, wt, b, act="silu")
    _check(O.Reference(x, 4, wt, b, 1e-5, "silu", dy), y, *_grads(y, (x, wt, b), dy))


@gpu
def test_an_outlier_in_the_first_place():
    dev = _dev()
    x = _map(1, 8, 40, 50, F32, dev=dev).clone(memory_format=torch.channels_last)
    x[:, :, 0, 0] = 1e4
    y = norm.group_norm_act(x, 2, act="none")
    _check(O.Reference(x, 2, None, None, 1e-5, "none"), y)


@gpu
def test_non_finite_values_stay_in_their_group():
    dev = _dev()
    x = _map(2, 12, 9, 11, F32, dev=dev).clone(memory_format=torch.channels_last)
    ref = norm.group_norm_act(x, 3)
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = x.clone(memory_format=torch.channels_last)
        z[1, 5, 3, 4] = bad  # group 1 of sample 1
        y = norm.group_norm_act(z, 3)
        assert y[1, 4:8].isnan().all()
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[1, 4:8] = False
        assert torch.equal(y[keep], ref[keep])


@gpu
def test_constant_group():
    """No spread: xhat = 0, y = act(bias), dx = 0 up to rstd = 1 / sqrt(eps)'s rounding."""
    dev = _dev()
    x = torch.full((2, 8, 5, 6), 3.25, device=dev).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    wt, b = _params(8, dev=dev)
    y = norm.group_norm_act(x, 2, wt, b)
    _check(O.Reference(x, 2, wt, b, 1e-5, "elu"), y)


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^32 values: the last sample is the one of a call of its own."""
    dev = _dev()
    n, c, h, w = 3, 32, 4096, 11008
    one = torch.randn(1, h, w, c, device=dev, dtype=BF16).permute(0, 3, 1, 2)
    wt, b = _params(c, dev=dev)
    x = one.expand(n, c, h, w).contiguous(memory_format=torch.channels_last)
    assert x.numel() > 2 ** 32
    y = norm.group_norm_act(x, 8, wt, b)
    # a sample's sums run over other parts in a smaller call: equal up to one rounding of bf16
    y1 = norm.group_norm_act(one, 8, wt, b)
    assert torch.equal(y[0], y[2])
    d = (y[2].float() - y1[0].float()).abs()
    assert (d <= 2 ** -7 * y1[0].float().abs() + 2 ** -20).all()
    del y, y1, d
    q = norm.act_checkpoint(x)
    assert torch.equal(q.q[-one.numel():], norm.act_checkpoint(one).q)
    assert torch.equal(norm.act_restore(q)[2], norm.act_restore(norm.act_checkpoint(one))[0])


# ------------------------------------------------------------------ 8-bit checkpoints
def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0), b.nan_to_num(0))


@gpu
@pytest.mark.parametrize("n", [1, 31, 32, 33, 1000, 8192, 100003])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_checkpoint_format(n, dtype):
    dev = _dev()
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g) * torch.exp(4 * torch.randn((n + 31) // 32, generator=g)).repeat_interleave(32)[:n]
    x[::7] = 0
    x = x.to(dtype).to(dev)
    c = norm.act_checkpoint(x)
    want, codes = O.through_8_bits(x.double())
    assert c.q.dtype == torch.int8 and c.q.shape == (n,) and c.scale.shape == ((n + 31) // 32,)
    assert torch.equal(c.scale.long(), codes) and c.nbytes() == n + (n + 31) // 32
    # (in fp16 some of these blocks hold an infinity: they restore as NaN)
    assert _same(norm.act_restore(c, F32).double(), want)  # exact in fp32
    assert _same(norm.act_restore(c), want.to(dtype))
    # 2^(code - 133) from its bits: a device pow is an ulp off, and ties are off by exactly half a step
    step = ((codes + (1023 - 133)) << 52).view(torch.float64).repeat_interleave(32)[:n]
    err, top = (want - x.double()).abs(), x.double().abs() > 126.5 * step
    assert (err <= torch.where(top, step, step / 2))[want.isfinite()].all()


@gpu
def test_checkpoint_extremes():
    """Zeros, subnormals, the largest values, ties, infinities and NaN, each in a block of its own."""
    dev = _dev()
    big = torch.finfo(F32).max
    rows = [[0.0], [-0.0], [1e-40, -1e-45], [2.0 ** -126, 2.0 ** -127], [big, -big, big / 2], [1.0, 0.5 / 64, 1.5 / 64,
            2.5 / 64], [127.5, -127.5, 0.5, 1.5], [float("inf"), 1.0], [1.0, -float("inf")], [float("nan"), 2.0], [65504.0]]
    x = torch.zeros(len(rows), 32)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
    x = x.to(dev)
    c = norm.act_checkpoint(x)
    want, codes = O.through_8_bits(x.reshape(-1).double())
    got = norm.act_restore(c, F32).reshape(-1)
    assert torch.equal(c.scale.long(), codes)
    assert _same(got.double(), want)
    assert codes.tolist().count(255) == 3
    half = norm.act_restore(norm.act_checkpoint(x[-1].half()))
    assert half.isfinite().all() and half[0] == 127 * 2.0 ** 9


@gpu
def test_checkpoint_keeps_layout():
    dev = _dev()
    x = _map(2, 12, 5, 7, F32, dev=dev)
    for t in (x, x.contiguous(), x.permute(2, 0, 3, 1), x[:, 2:9], x[0, 0, 0, 0], x[:1, :1].expand(3, 4, 5, 7)):
        r = norm.act_restore(norm.act_checkpoint(t))
        assert r.shape == t.shape and r.dtype == t.dtype
        assert ((r - t).abs() <= t.abs().max() / 64).all()
    assert norm.act_restore(norm.act_checkpoint(x)).stride() == x.stride()
    store = torch.zeros(65, device=dev)
    store[1:] = torch.randn(64, device=dev)
    off = store[1:]
    assert off.data_ptr() % 16 and torch.equal(norm.act_checkpoint(off).q, norm.act_checkpoint(off.clone()).q)


@pytest.mark.skip(reason="an illegal address after the solver's tests in one process, cause unknown: the library's "
                         "convolution gradients and 64-bit products stay off (test_norm_encoder.py)")
@gpu
@pytest.mark.parametrize("cl", [False, True])
def test_conv2d_from_a_checkpoint(cl):
    """y and dx are the library's own; the weight's gradient is the library's at the restored input."""
    dev = _dev()
    x = _map(2, 8, 14, 18, F32, dev=dev)
    x = (x if cl else x.contiguous()).requires_grad_(True)
    wt = (0.1 * torch.randn(12, 8, 1, 1, generator=torch.Generator().manual_seed(1))).to(dev).requires_grad_(True)
    b = torch.zeros(12, device=dev, requires_grad=True)
    dy = _map(2, 12, 14, 18, F32, seed=2, dev=dev)
    y = norm.conv2d(x, wt, b)
    dx, dw, db = _grads(y, (x, wt, b), dy)
    xr = O.through_8_bits((x.permute(0, 2, 3, 1) if cl else x).detach().reshape(-1).double())[0]
    xr = xr.view(2, 14, 18, 8).permute(0, 3, 1, 2) if cl else xr.view(2, 8, 14, 18)
    d64, w64, x64 = dy.double(), wt.detach().double()[:, :, 0, 0], x.detach().double()
    # 504 products to a weight's gradient, 8 to a value of y, 12 to one of dx, in an order of the library's own
    for got, f, terms in ((dw[:, :, 0, 0], lambda a, c, i: torch.einsum("nohw,nihw->oi", a, i), 504),
                          (y, lambda a, c, i: torch.einsum("oi,nihw->nohw", c, x64 if i is xr else x64.abs()), 9),
                          (dx, lambda a, c, i: torch.einsum("oi,nohw->nihw", c, a), 12)):
        ref, mag = f(d64, w64, xr), f(d64.abs(), w64.abs(), xr.abs())
        assert ((got.double() - ref).abs() <= terms * O.U * mag).all()
    assert ((db.double() - d64.sum((0, 2, 3))).abs() <= 504 * O.U * d64.abs().sum((0, 2, 3))).all()


@gpu
@pytest.mark.parametrize("cl", [False, True])
@pytest.mark.parametrize("autocast", [False, True])
def test_conv2d_gives_the_restored_input(cl, autocast, monkeypatch):
    """What the convolution's backward pass is given, recorded in place of the library's: dy, the restored x in
    x's own layout, the convolution's numbers; y is the convolution's (which runs on the CPU)."""
    dev = _dev()
    x = _map(2, 8, 14, 18, F32, dev=dev)
    x = (x if cl else x.contiguous()).requires_grad_(True)
    wt = (0.1 * torch.randn(12, 4, 3, 3, generator=torch.Generator().manual_seed(1))).to(dev).requires_grad_(True)
    b = torch.zeros(12, device=dev, requires_grad=True)
    given, ys, plain = [], [], torch.nn.functional.conv2d

    def conv(x, weight, bias, *a):
        ys.append(plain(x.cpu(), weight.cpu(), bias.cpu(), *a).to(dev))
        return ys[-1]

    def backward(g, xb, weight, *a):
        given.append((g, xb, a))
        return torch.ones_like(xb), torch.full_like(weight, 2), torch.full((12,), 3, dtype=xb.dtype, device=dev)
    monkeypatch.setattr(torch.nn.functional, "conv2d", conv)
    monkeypatch.setattr(norm, "_convolution_backward", backward)
    with torch.autocast("cuda", dtype=BF16, enabled=autocast):
        y = norm.conv2d(x, wt, b, 2, (1, 2), dilation=2, groups=2)
    t = BF16 if autocast else F32
    assert y.dtype == t and torch.equal(y, ys[0])
    dy = torch.randn(y.shape, device=dev, dtype=t)
    dx, dw, db = _grads(y, (x, wt, b), dy)
    (g, xb, a), = given
    want = norm.act_restore(norm.act_checkpoint(x.detach().to(t)))
    assert torch.equal(g, dy) and torch.equal(xb, want) and xb.dtype == t and xb.stride() == x.stride()
    assert a == ([12], [2, 2], [1, 2], [2, 2], False, [0, 0], 2, [True, True, True])
    assert (dx == 1).all() and (dw == 2).all() and (db == 3).all()
    assert dx.dtype == dw.dtype == db.dtype == F32  # the leaves' own
    with pytest.raises(ValueError):
        norm.conv2d(x[0], wt, b, 2, (1, 2), dilation=2, groups=2)
    del given[:]
    z = norm.conv2d(x, wt.detach(), b, 2, (1, 2), dilation=2, groups=2)  # no gradient of the weight: nothing kept
    assert z.requires_grad and "Checkpoint" not in type(z.grad_fn).__name__ and not given


# ------------------------------------------------------------------ as torch operators
@gpu
def test_compiled_call_is_the_eager_one():
    """Traced without a graph break, forward and backward: the eager call's bits."""
    dev = _dev()
    wt, b = (p.requires_grad_(True) for p in _params(16, dev=dev))
    dy = _map(2, 16, 9, 11, F32, seed=7, dev=dev)

    def block(x, ck):
        return norm.group_norm_act(x * 2, 4, wt, b, act="silu", checkpoint=ck) + 1
    for ck in (False, True):
        x = _map(2, 16, 9, 11, F32, dev=dev).requires_grad_(True)
        fast = torch.compile(block, backend="aot_eager", fullgraph=True)
        y, z = block(x, ck), fast(x, ck)
        assert torch.equal(y, z)
        for u, v in zip(_grads(y, (x, wt, b), dy), _grads(z, (x, wt, b), dy)):
            assert torch.equal(u, v)
        for h, w in ((7, 20), (5, 4)):  # other sizes, which then are symbols
            x = _map(3, 16, h, w, F32, dev=dev).requires_grad_(True)
            assert torch.equal(block(x, ck), fast(x, ck))


@gpu
def test_gradients_once_twice_and_shared():
    """The same graph twice, one tensor as weight and bias, two calls on one x; not a gradient's gradient."""
    dev = _dev()
    x = _map(2, 16, 9, 11, F32, dev=dev).requires_grad_(True)
    wt, b = (p.requires_grad_(True) for p in _params(16, dev=dev))
    dy = _map(2, 16, 9, 11, F32, seed=7, dev=dev)
    y = norm.group_norm_act(x, 4, wt, b)
    one = torch.autograd.grad(y, (x, wt, b), dy, retain_graph=True)
    two = torch.autograd.grad(y, (x, wt, b), dy, retain_graph=True)
    assert all(torch.equal(u, v) for u, v in zip(one, two))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y, x, dy, create_graph=True)
    both, = torch.autograd.grad(norm.group_norm_act(x, 4, wt, wt), wt, dy)
    v, c = wt.detach().clone().requires_grad_(True), wt.detach().clone().requires_grad_(True)
    dv, dc = torch.autograd.grad(norm.group_norm_act(x, 4, v, c), (v, c), dy)
    assert torch.equal(both, dv + dc)
    dx, = torch.autograd.grad(y + norm.group_norm_act(x, 4, wt, b), x, dy)
    assert torch.equal(dx, one[0] + one[0])


@gpu
def test_operator_refuses_what_does_not_belong_together():
    dev = _dev()
    x = _map(2, 16, 9, 11, F32, dev=dev)
    wt, b = _params(16, dev=dev)
    ops = N.torch_ops()
    none = torch.empty(0, device=dev)
    y, stat, q, scale = ops.group_norm_act_forward(x, 4, wt, b, 1e-5, 2, False, True, True)
    good = dict(dy=x, x=x, q=none, scale=none, weight=wt, bias=b, stat=stat, groups=4, eps=1e-5, act=2, need_x=True,
                need_w=True, need_b=True)
    ops.group_norm_act_backward(**good)
    half = x.to(BF16)
    for bad in (dict(x=none), dict(x=x[:1]), dict(x=half), dict(q=q, scale=scale), dict(x=none, q=q),
                dict(x=none, q=q[1:], scale=scale), dict(x=none, q=q[::2], scale=scale), dict(stat=stat[:1]),
                dict(stat=stat.double()), dict(weight=None), dict(bias=None), dict(groups=2), dict(groups=3),
                dict(weight=wt[:8]), dict(stat=stat.cpu()), dict(x=x.cpu())):
        with pytest.raises(ValueError):
            ops.group_norm_act_backward(**{**good, **bad})
    c = norm.act_checkpoint(x)
    for bad in ((c.q[1:], c.scale, c.shape, c.stride), (c.q, c.scale[1:], c.shape, c.stride), (c.q, c.scale, c.shape, (0, 1, 1, 1)),
                (c.q.float(), c.scale, c.shape, c.stride), (c.q, c.scale.cpu(), c.shape, c.stride)):
        with pytest.raises(ValueError):
            norm.act_restore(norm.ActCheckpoint(*bad, F32))
    with pytest.raises(TypeError):
        norm.act_restore(c, torch.float64)
    with pytest.raises(ValueError):
        norm.group_norm_act(x, 4, wt.cpu())


# ------------------------------------------------------------------ streams, graphs, repeats
@gpu
def test_runs_are_bit_identical_and_streams_share_nothing():
    dev = _dev()
    xs = [_map(4, 32, 60, 80, F32, seed=i, dev=dev).requires_grad_(True) for i in range(4)]
    wt, b = (p.requires_grad_(True) for p in _params(32, dev=dev))
    dy = _map(4, 32, 60, 80, F32, seed=9, dev=dev)

    def step(x):
        y = norm.group_norm_act(x, 8, wt, b, checkpoint=True)
        return (y.detach(),) + _grads(y, (x, wt, b), dy)
    ref = [step(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    outs = []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(step(x))
    torch.cuda.synchronize()
    for a, r in zip(outs, ref):
        assert all(torch.equal(u, v) for u, v in zip(a, r))


@gpu
def test_two_threads_at_once():
    """Calls from two host threads, each on a stream of its own, and in inference mode."""
    import threading
    dev = _dev()
    wt, b = _params(24, dev=dev)
    xs = [_map(2, 24, 40, 50, F32, seed=i, dev=dev) for i in range(2)]
    ref = [norm.group_norm_act(x, 6, wt, b) for x in xs]
    with torch.inference_mode():
        assert torch.equal(norm.group_norm_act(xs[0], 6, wt, b), ref[0])
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[i].append(norm.group_norm_act(xs[i], 6, wt, b))
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(len(g) == 20 and all(torch.equal(y, r) for y in g) for g, r in zip(got, ref))


@gpu
def test_captured_step_replays():
    """A forward and backward pass in one graph, replayed on new contents between eager calls; two
    graphs of one stream share nothing, replayed side by side."""
    dev = _dev()
    wt, b = (p.requires_grad_(True) for p in _params(16, dev=dev))
    dy = _map(2, 16, 30, 40, F32, seed=7, dev=dev)
    ins = [_map(2, 16, 30, 40, F32, seed=i, dev=dev).clone(memory_format=torch.channels_last).requires_grad_(True)
           for i in range(2)]

    def step(x):
        y = norm.group_norm_act(x, 4, wt, b, act="silu", checkpoint=True)
        return (y.detach(),) + _grads(y, (x, wt, b), dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(ins[0])
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(step(x))
        graphs.append(g)
    side = torch.cuda.Stream()
    for rep in range(4):
        fresh = [_map(2, 16, 30, 40, F32, seed=20 + 2 * rep + i, dev=dev) for i in range(2)]
        with torch.no_grad():
            for x, f in zip(ins, fresh):
                x.copy_(f)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for f, o in zip(fresh, outs):
            want = step(f.detach().requires_grad_(True))
            assert all(torch.equal(u, v) for u, v in zip(o, want)), rep
