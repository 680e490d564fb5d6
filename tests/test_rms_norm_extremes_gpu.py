"""Root-mean-square norm of finite rows whose squares leave fp32's range, against the definition in 64 bits (tests/blocks_ref.py).

Tolerances: those of tests/test_rms_norm_gpu.py -- S = H / 64 + 16 steps of u = 2^-24 for the sum (a power of two before it changes none of them), (S / 2 + 6) u of |y| --, and
half a step of the type's subnormals where a result may lie there: 2^-150 (f32), 2^-134 (bf16), a few of them for dx's three roundings."""
import pytest
import torch

import blocks_ref as ref
import strict

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
WIDTHS = [1, 5, 32, 40, 100, 128, 200, 256, 300, 768, 1001, 1536, 2000, 2304, 5001, 8192, 16384]      # every number of lanes per row


def _ops():
    from merlot_amd import ops
    return ops


def _rows(H, dtype, size, seed):
    """rows of magnitude `size` between ordinary ones (neighbours in a wave take the other way)"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(7, H, generator=g).clamp(-2.5, 2.5)
    x[x.abs() < 0.01] = 0.5
    x[1::2] *= size
    return x.to(dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('H', WIDTHS)
@pytest.mark.parametrize('size,eps', [(1e30, 1e-6), (2e19, 1e-6), (1e37, 1e-6), (1e-25, 0.0), (1e-30, 0.0), (1e-25, 1e-45), (1e-25, 3e-38), (1e-20, 1e-36)])
def test_forward_and_backward(H, dtype, size, eps):
    ops = _ops()
    eps = float(torch.tensor(eps))                             # the value that the kernel gets
    x, gamma = _rows(H, dtype, size, H), 1.0 + 0.2 * torch.randn(H, generator=torch.Generator().manual_seed(H))
    res = _rows(H, dtype, size, H + 1)
    for r in (None, res):
        hr, yr, rr = ref.rms(x, r, gamma, eps)
        assert bool(torch.isfinite(hr.double()).all()) and bool((rr < 2.0 ** 127).all()) and bool((rr > 2.0 ** -126).all())
        steps = (H / 64 + 16) / 2 + 6
        y, h, rstd, y8, s8 = ops.rms_norm_fwd(x.cuda(), gamma.cuda(), residual=None if r is None else r.cuda(), q8=True, eps=eps)
        assert r is None or torch.equal(h.cpu(), hr)
        strict.close(y, yr, yr.abs() * (steps * U + HALF[dtype]) + 2 * TINY[dtype], 'y')
        strict.close(rstd, rr[:, 0], rr[:, 0] * steps * U, 'rstd')
        alone = ops.rms_norm_fwd(x.cuda(), gamma.cuda(), residual=None if r is None else r.cuda(), eps=eps)
        strict.close(alone[0], yr, yr.abs() * (steps * U + HALF[dtype]) + 2 * TINY[dtype], 'y without the 8-bit copy')
        strict.close(alone[2], rr[:, 0], rr[:, 0] * steps * U, 'rstd without the 8-bit copy')
        # half a step of e4m3, 2^-4 of the value or of the least normals' step under the larger of the two scales that a maximum next to a border may take
        pad = torch.nn.functional.pad(yr, (0, y8.shape[1] - H)).view(7, -1, 128).abs().amax(-1)
        unit = ref.pow2(ref.exponents(pad, 0) + 1 - 10).repeat_interleave(128, 1)[:, :H]
        got = ref.values(y8, s8)
        strict.close(got[:, :H], yr, torch.maximum(yr.abs() * 2.0 ** -4, unit) * (1 + 2.0 ** -10) + yr.abs() * steps * U, 'y8')
        # (h near 1e-30 with a gradient of order 1 would have a dx over 1e30 that is right but says little: the gradient is taken at the row's own size)
        dy = _rows(H, dtype, 1.0, H + 2)
        dgamma = torch.zeros(H, device='cuda')
        dx = ops.rms_norm_bwd(dy.cuda(), x.cuda() if r is None else h, rstd, gamma.cuda(), dgamma)
        dxr, dgr = ref.rms_bwd(dy, hr, gamma, eps)
        n, t = hr.double() * rr, dy.double() * gamma.double()
        scale = rr * (t.abs() + n.abs() * (t * n).abs().mean(-1, keepdim=True))
        strict.close(dx, dxr, scale * (H / 64 + 32) * U + dxr.abs() * (HALF[dtype] + 2 * U) + 8 * TINY[dtype], 'dx')
        strict.close(dgamma, dgr, (dy.double() * n).abs().sum(0) * (steps + 30) * U + 8 * TINY[torch.float32], 'dgamma')


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_the_ends_of_the_range(dtype):
    """the type's largest values; one element over 2^64 alone; subnormals with no eps, whose 1 / rms is over fp32's range (y is not); rows of zeros"""
    ops = _ops()
    for H in (1, 33, 100, 300, 1000, 2304, 16384):
        x = torch.zeros(6, H, dtype=dtype)
        x[0] = torch.finfo(dtype).max
        x[1, H // 2] = 2.5e19
        x[2] = 2.0 ** -126
        x[3] = 2.0 ** -133                                     # (subnormal in both types)
        x[4] = 1.0
        gamma = torch.linspace(0.5, 1.5, H)
        steps = (H / 64 + 16) / 2 + 6
        y, _, rstd, _, _ = ops.rms_norm_fwd(x.cuda(), gamma.cuda(), eps=0.0)
        _, yr, rr = ref.rms(x[:5], None, gamma, 0.0)
        strict.close(y[:5], yr, yr.abs() * (steps * U + HALF[dtype]) + 2 * TINY[dtype], H)
        # the largest values: R under 2^-126 is rounded to 2^-149 (half a step: 2^-150)
        strict.close(rstd[[0, 1, 2, 4]], rr[[0, 1, 2, 4], 0], rr[[0, 1, 2, 4], 0] * steps * U + 2.0 ** -150, H)
        assert float(rstd[3]) == float('inf') and bool(torch.isnan(y[5]).all()) and float(rstd[5]) == float('inf')      # 0 / 0, as the definition has it
        y, _, rstd, _, _ = ops.rms_norm_fwd(x.cuda(), gamma.cuda(), eps=1e-30)
        _, yr, rr = ref.rms(x, None, gamma, float(torch.tensor(1e-30)))
        strict.close(y, yr, yr.abs() * (steps * U + HALF[dtype]) + 2 * TINY[dtype], H)
        strict.close(rstd, rr[:, 0], rr[:, 0] * steps * U + 2.0 ** -150, H)
