"""Group normalisation with an activation, its gradients and the 8-bit checkpoint in 64 bits, from
their formulas, with the bounds that fp32 arithmetic and one rounding to the values' type set."""
import torch

U = 2.0 ** -24  # half a step of fp32


def act(z, name):
    if name == "elu":
        return torch.where(z > 0, z, torch.expm1(z.clamp(max=0)))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    return z


def slope(z, name):
    if name == "elu":
        return torch.exp(z.clamp(max=0))
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "relu":
        return (z > 0).to(z.dtype)
    return torch.ones_like(z)


def through_8_bits(flat):
    """flat (64 bits) -> (restored, scale codes): blocks of 32, step 2^(E - 133) with E the biased
    fp32 exponent of the block's largest magnitude, clamped to [7, 254]; NaN for a block that is not
    finite (255)."""
    n = flat.numel()
    v = torch.zeros(-(-n // 32) * 32, dtype=torch.float64, device=flat.device)
    v[:n] = flat.double()
    v = v.view(-1, 32)
    bad = ~torch.isfinite(v).all(1)
    top = torch.where(bad, torch.ones_like(v[:, 0]), v.abs().amax(1))
    e = torch.frexp(top)[1].long() - 1  # 2^e <= top < 2^(e + 1)
    e = torch.where(top > 0, e, torch.full_like(e, -1000)).clamp(-120, 127)
    step = ((1023 + e - 6) << 52).view(torch.float64)[:, None]
    q = (v / step).round().clamp(-127, 127) * step
    q[bad] = float("nan")
    return q.view(-1)[:n], torch.where(bad, torch.full_like(e, 255), e + 127)


class Reference:
    """Everything in fp64, NCHW: y, and with dy dx, dweight, dbias; *_tol the bounds.

    The bounds: mean and rstd come from sums of at most `run` terms in a row in fp32 (a thread's) and
    fp64 above that: off by (run + 8) U of the terms' magnitudes.  z takes three roundings more, an
    activation 8 U of its value (its exponential and reciprocal are within 2 U each) and a slope of at
    most 1.1; a stored value half a step of its type.  The ELU of a 16-bit map is expm1 to z^3 above
    -1/16: the next term is z^4 / 24 of a value of at least |z| (1 - |z| / 2), so 2^-12 / 24 x 32 / 31 =
    2^-16.5 of it; below, the exponential's 2 U become at most 2 U x 16 = 2^-19 of the value."""

    def __init__(self, x, groups, weight, bias, eps, name, dy=None, checkpoint=False, run=64):
        n, c, h, w = x.shape
        t = x.dtype
        half = torch.finfo(t).eps / 2
        tiny = torch.finfo(t).tiny * torch.finfo(t).eps if t != torch.float32 else 0.0  # subnormal steps
        x = x.detach().double()
        g = torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.detach().double()
        b = torch.zeros(c, dtype=torch.float64, device=x.device) if bias is None else bias.detach().double()
        g, b = g.view(1, c, 1, 1), b.view(1, c, 1, 1)
        d = c // groups

        def gmean(v):
            m = v.reshape(n, groups, -1).mean(2)
            return m.repeat_interleave(d, 1).view(n, c, 1, 1)

        mean = gmean(x)
        var = gmean((x - mean) ** 2)
        rstd = (var + eps).rsqrt()
        mean_tol = (run + 8) * U * gmean((x - mean).abs()) + 4 * U * mean.abs()
        rstd_rel = (run + 8) * U
        self.mean, self.rstd = mean.view(n, c)[:, ::d], rstd.view(n, c)[:, ::d]

        def z_of(v):
            xhat = (v - mean) * rstd
            xhat_tol = xhat.abs() * (rstd_rel + 4 * U) + rstd * (mean_tol + 2 * U * mean.abs())
            return xhat, xhat_tol, xhat * g + b, xhat_tol * g.abs() + 2 * U * (xhat * g).abs() + 2 * U * b.abs()

        xhat, xhat_tol, z, z_tol = z_of(x)
        self.z, self.z_tol = z, z_tol
        self.y = act(z, name)
        y32 = 1.1 * z_tol + (8 * U + (2.0 ** -16.5 if name == "elu" and t != torch.float32 else 0.0)) * self.y.abs()
        self.y_tol = y32 + half * (self.y.abs() + y32) + tiny
        if dy is None:
            return
        if checkpoint:
            flat = x.permute(0, 2, 3, 1).reshape(-1)
            x = through_8_bits(flat)[0].view(n, h, w, c).permute(0, 3, 1, 2)
            xhat, xhat_tol, z, z_tol = z_of(x)
        dy = dy.double()
        k = slope(z, name)
        u = dy * k
        u_tol = dy.abs() * (z_tol if name in ("elu", "silu") else 0 * z_tol) + 8 * U * u.abs()
        self.dbias, self.dweight = u.sum((0, 2, 3)), (u * xhat).sum((0, 2, 3))
        one = (run + 8) * U
        self.dbias_tol = (u_tol + one * u.abs()).sum((0, 2, 3))
        w_tol = u_tol * xhat.abs() + u.abs() * xhat_tol + one * (u * xhat).abs()
        self.dweight_tol = w_tol.sum((0, 2, 3))
        m1, m2 = gmean(g * u), gmean(g * u * xhat)
        m1_tol = gmean(g.abs() * (u_tol + one * u.abs()))
        m2_tol = gmean(g.abs() * w_tol)
        self.dx = rstd * (g * u - m1 - xhat * m2)
        parts = rstd * ((g * u).abs() + m1.abs() + (xhat * m2).abs())
        dx32 = (rstd_rel * 3 + 8 * U) * parts + rstd * (g.abs() * u_tol + m1_tol + xhat.abs() * m2_tol
                                                        + xhat_tol * m2.abs())
        self.dx_tol = dx32 + half * (self.dx.abs() + dx32) + tiny


def excess(got, want, tol):
    """max(|got - want| - tol): not positive where every value is within its bound."""
    return float(((got.detach().double() - want.detach()).abs() - tol.detach()).max()) if want.numel() else 0.0
