"""TEST-ONLY definitions of the root-mean-square norm, the 8-bit blocks and the gradient clip in plain torch, 64 bits, on the CPU."""
import torch

FORMATS = {0: (torch.float8_e4m3fn, 8, 3, -6), 1: (torch.float8_e5m2, 15, 2, -14)}      # dtype, largest = 1.75 * 2^top, mantissa bits, least normal exponent


def pow2(e):
    """2^e in 64 bits, exactly"""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exponents(amax, fmt):
    """amax f64 -> the least e >= -127 with amax <= 1.75 * 2^(top + e); 0 for zeros"""
    top = FORMATS[fmt][1]
    m, p = torch.frexp(amax)                               # amax = m * 2^p, m in [0.5, 1)
    e = (p.long() - 1 - top + (m > 0.875).long()).clamp(min=-127)
    return torch.where(amax == 0, torch.zeros_like(e), e)


def quantize(x, fmt, tile=1):
    """x [R, C] -> (codes as float8 [R, Cp], scale bytes [R, Cp / 128], values f64 [R, Cp])"""
    dt, top, mant, low = FORMATS[fmt]
    x = x.double()
    R, C = x.shape
    Cp = (C + 127) // 128 * 128
    xp = torch.zeros((R, Cp), dtype=torch.float64)
    xp[:, :C] = x
    b = xp.view(R, Cp // 128, 128)
    bad = ~torch.isfinite(b).all(-1)
    amax = torch.nan_to_num(b, nan=0.0, posinf=0.0, neginf=0.0).abs().amax(-1)
    if tile == 128:
        for r in range(0, R, 128):
            amax[r:r + 128] = amax[r:r + 128].amax(0, keepdim=True)
            bad[r:r + 128] = bad[r:r + 128].any(0, keepdim=True)
    e = exponents(amax, fmt)
    u = b * pow2(-e).unsqueeze(-1)
    _, p = torch.frexp(torch.nan_to_num(u, nan=0.0, posinf=0.0, neginf=0.0).abs().clamp(min=2.0 ** low))
    step = pow2(p.long() - 1 - mant)
    v = torch.round(u / step) * step                       # torch.round: ties to even
    v = torch.where(bad.unsqueeze(-1), torch.full_like(v, float('nan')), v)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return v.view(R, Cp).float().to(dt), byte, (v * pow2(e).unsqueeze(-1)).view(R, Cp)


def values(q, s):
    """codes + scale bytes -> f64 values"""
    q, s = q.cpu(), s.cpu()
    sc = torch.where(s == 255, torch.full(s.shape, float('nan'), dtype=torch.float64), pow2(s.long() - 127))
    return (q.double().view(q.shape[0], -1, 128) * sc.unsqueeze(-1)).view(q.shape)


def rms(x, res, gamma, eps):
    """-> h (in x's type), y f64, rstd f64"""
    h = x if res is None else (x.double() + res.double()).to(x.dtype)
    hd = h.double()
    rstd = 1.0 / torch.sqrt(hd.pow(2).mean(-1, keepdim=True) + eps)
    return h, hd * rstd * gamma.double(), rstd


def rms_bwd(dy, h, gamma, eps, dres=None):
    hd, dy, g = h.double(), dy.double(), gamma.double()
    rstd = 1.0 / torch.sqrt(hd.pow(2).mean(-1, keepdim=True) + eps)
    n = hd * rstd
    t = dy * g
    dx = rstd * (t - n * (t * n).mean(-1, keepdim=True))
    return (dx if dres is None else dx + dres.double()), (dy * n).sum(0)
