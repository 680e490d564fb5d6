"""Root-mean-square norm (merlot_rms_fwd / merlot_rms_bwd, layers.rms_norm) against its definition in 64 bits (tests/blocks_ref.py).

Tolerances, per element.  u = 2^-24 (fp32, half a step).  The sum of H squares in fp32, in any order: relative error at most (H + 2) u, here far fewer rounding steps (a
lane adds at most H / 64 + 1 values, then 6 + 4 joins): S = H / 64 + 16 steps; 1 / sqrt halves it and adds 3 roundings, the two products 2 more: (S / 2 + 6) u of |y|.
The output's own rounding: half a step of its type, 2^-8 (bf16) or u (f32) of the value."""
import pytest
import torch

import blocks_ref as ref

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
U = 2.0 ** -24
EPS = 1e-6


def _ops():
    from merlot_amd import ops
    return ops


def _data(rows, H, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, H + pad, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    x[:, ::37] *= 15.0
    return x.to(dtype)


def _strided(x, H):
    return x.cuda()[:, :H]


def _close(got, want, tol, what):
    bad = (got.double().cpu() - want).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double().cpu() - want).abs() / tol.clamp(min=1e-300)).max()))


# every (elements per lane, slabs, lanes per row) variant, its first and last width, odd widths, and views whose rows are 2- or 4-byte aligned only
WIDTHS = [1, 2, 7, 8, 9, 16, 31, 32, 33, 63, 64, 65, 100, 127, 128, 130, 255, 256, 257, 500, 512, 768, 769, 1000, 1001, 1024, 1025, 1531, 1536, 1537, 2047, 2048, 2049, 4096, 4100, 5001,
          6144, 6145, 8192, 8200, 16384]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('H', WIDTHS)
def test_forward_and_backward(H, dtype):
    ops = _ops()
    for rows, pad, with_res in ((1, 0, True), (5, 3, False), (67, 8, True)):
        x = _data(rows, H, dtype, H + rows, pad)
        res = _data(rows, H, dtype, H + rows + 1) if with_res else None
        gamma = 1.0 + 0.2 * torch.randn(H, generator=torch.Generator().manual_seed(H))
        xg = _strided(x, H)
        y, h, rstd, y8, s8 = ops.rms_norm_fwd(xg, gamma.cuda(), residual=None if res is None else res.cuda(), q8=True, eps=EPS)
        hr, yr, rr = ref.rms(x[:, :H], res, gamma, EPS)
        if with_res:
            assert torch.equal(h.cpu(), hr)
        else:
            assert h is None
        steps = (H / 64 + 16) / 2 + 6
        _close(y, yr, yr.abs() * (steps * U + HALF[dtype]) + 1e-40, 'y')
        _close(rstd, rr[:, 0], rr[:, 0] * steps * U, 'rstd')
        alone = ops.rms_norm_fwd(xg, gamma.cuda(), residual=None if res is None else res.cuda(), eps=EPS)      # narrow rows: fewer lanes each without the 8-bit copy
        _close(alone[0], yr, yr.abs() * (steps * U + HALF[dtype]) + 1e-40, 'y alone')
        _close(alone[2], rr[:, 0], rr[:, 0] * steps * U, 'rstd alone')
        assert h is None or torch.equal(alone[1], h)
        # the 8-bit copy of the unrounded y: half a step of e4m3 (2^-4 of the value, or of the least normal 2^-6 of the block's unit) beside y's own error; a block whose
        # maximum lies within y's error of a border of the scale may take the neighbouring power of two, whose half steps are twice as large only below the normal range
        _, _, v = ref.quantize(yr, 0)
        got = ref.values(y8, s8)
        e = ref.exponents(torch.nn.functional.pad(yr, (0, got.shape[1] - H)).view(rows, -1, 128).abs().amax(-1), 0)
        unit = ref.pow2(e + 1 - 10).repeat_interleave(128, 1)[:, :H]        # half a step of the least normals, under the larger of the two possible scales
        _close(got[:, :H], yr, torch.maximum(yr.abs() * 2.0 ** -4, unit) * (1 + 2.0 ** -10) + yr.abs() * steps * U, 'y8')
        assert float(got[:, H:].abs().sum()) == 0.0 and s8.shape == (rows, got.shape[1] // 128)
        assert float((got[:, :H] != v[:, :H]).double().mean()) < 0.02 or rows * H < 200       # the same rounding but for values next to a tie

        dy, dres = _data(rows, H, dtype, H + rows + 2), _data(rows, H, dtype, H + rows + 3)
        hin = h if with_res else xg
        dgamma = torch.full((H,), 0.5, device='cuda')
        dx = ops.rms_norm_bwd(dy.cuda(), hin, rstd, gamma.cuda(), dgamma, dres=dres.cuda())
        dxr, dgr = ref.rms_bwd(dy, hr, gamma, EPS, dres)
        # dx = R (t - n c): t with 1 rounding, n 1 + R's, c a sum of H terms each |t n| -> absolute error under R * (|t| + |n| mean|t n|) * (steps + 8) u, + dres, + the store
        n = hr.double() * rr
        t = dy.double() * gamma.double()
        scale = rr * (t.abs() + n.abs() * (t * n).abs().mean(-1, keepdim=True))
        _close(dx, dxr, scale * (H / 64 + 32) * U + (dxr.abs() + dres.double().abs()) * (HALF[dtype] + 2 * U) + 1e-40, 'dx')
        # dgamma: rows + 20 additions of terms with `steps` roundings each, on top of 0.5
        _close(dgamma, dgr + 0.5, (dy.double() * n).abs().sum(0) * (steps + rows + 20) * U + 4 * U * (dgr.abs() + 0.5), 'dgamma')
        again = torch.full((H,), 0.5, device='cuda')
        dx2 = ops.rms_norm_bwd(dy.cuda(), hin, rstd, gamma.cuda(), again, dres=dres.cuda())
        assert torch.equal(dx2, dx) and torch.equal(again, dgamma)             # no atomics: the same bits


def test_many_rows_take_every_loop_iteration():
    """more rows than workgroups: the grid-stride loops and the partial sums of dgamma"""
    ops = _ops()
    for rows, H in ((20011, 256), (9001, 768), (5003, 2304)):
        x = _data(rows, H, torch.float32, rows)
        gamma = torch.linspace(0.5, 1.5, H)
        y, _, rstd, _, _ = ops.rms_norm_fwd(x.cuda(), gamma.cuda(), eps=EPS)
        _, yr, rr = ref.rms(x, None, gamma, EPS)
        _close(y, yr, yr.abs() * ((H / 64 + 16) / 2 + 7) * U + 1e-40, 'y')
        dy = _data(rows, H, torch.float32, rows + 1)
        dgamma = torch.zeros(H, device='cuda')
        dx = ops.rms_norm_bwd(dy.cuda(), x.cuda(), rstd, gamma.cuda(), dgamma)
        dxr, dgr = ref.rms_bwd(dy, x, gamma, EPS)
        n, t = x.double() * rr, dy.double() * gamma.double()
        _close(dx, dxr, rr * (t.abs() + n.abs() * (t * n).abs().mean(-1, keepdim=True)) * (H / 64 + 32) * U + 1e-40, 'dx')
        # a lane adds at most rows / 4096 + 1 rows (4 096 row slots at most), then 4 + 1024 / 16 + 16 joins; 40 more for the terms themselves
        _close(dgamma, dgr, (dy.double() * n).abs().sum(0) * (rows / 1024 + 130 + H / 128) * U, 'dgamma')


def test_zeros_extremes_and_rows_that_are_not_finite():
    ops = _ops()
    H = 300
    for dtype in (torch.bfloat16, torch.float32):
        x = _data(6, H, dtype, 3)
        x[0] = 0
        x[1, 5] = float('inf')
        x[2, 7] = float('nan')
        x[3] = 1e-30
        gamma = torch.ones(H)
        y, _, rstd, y8, s8 = ops.rms_norm_fwd(x.cuda(), gamma.cuda(), q8=True, eps=EPS)
        y, v = y.float().cpu(), ref.values(y8, s8)
        assert bool((y[0] == 0).all()) and bool((v[0] == 0).all()) and abs(float(rstd[0]) - 1e3) < 1e-3
        assert bool(torch.isnan(y[1, 5])) and bool((y[1, :5] == 0).all())      # inf * 0 where the row's infinity stands, 0 elsewhere
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(v[2]).all())
        assert bool(torch.isnan(v[1, :128]).all()) and bool((v[1, 128:] == 0).all())
        _, yr, _ = ref.rms(x, None, gamma, EPS)
        for r in (3, 4, 5):
            _close(y[r], yr[r], yr[r].abs() * (16 * U + HALF[dtype]) + 1e-40, r)


def test_no_rows_and_leading_dimensions():
    ops = _ops()
    gamma = torch.ones(96, device='cuda')
    y, h, rstd, y8, s8 = ops.rms_norm_fwd(torch.empty(0, 96, device='cuda'), gamma, q8=True)
    assert y.shape == (0, 96) and rstd.shape == (0,) and y8.shape == (0, 128)
    dg = torch.ones(96, device='cuda')
    assert ops.rms_norm_bwd(y, y, rstd, gamma, dg).shape == (0, 96) and bool((dg == 1).all())
    x = torch.randn(3, 4, 96, device='cuda')
    y = ops.rms_norm_fwd(x, gamma)[0]
    assert y.shape == x.shape and torch.equal(y.view(-1, 96), ops.rms_norm_fwd(x.view(-1, 96), gamma)[0])


def test_layer_gradients_against_differences():
    """layers.rms_norm: the gradients of x, the residual and the gain against central differences of the 64-bit definition, and both outputs used"""
    from merlot_amd import layers

    class Norm(object):
        pass
    H, rows = 40, 3
    g = torch.Generator().manual_seed(11)
    x, r = torch.randn(rows, H, generator=g), torch.randn(rows, H, generator=g)
    wy, wh = torch.randn(rows, H, generator=g), torch.randn(rows, H, generator=g)
    norm = Norm()
    norm.gamma, norm.ggamma = (1 + 0.3 * torch.randn(H, generator=g)).cuda(), torch.zeros(H, device='cuda')
    xg, rg = x.cuda().requires_grad_(), r.cuda().requires_grad_()
    y, h = layers.rms_norm(xg, norm, residual=rg, eps=EPS)
    ((y * wy.cuda()).sum() + (h * wh.cuda()).sum()).backward()

    def loss(xx, gg):
        hh = xx + r.double()
        return float(((hh / torch.sqrt(hh.pow(2).mean(-1, keepdim=True) + EPS) * gg) * wy.double()).sum() + (hh * wh.double()).sum())
    gam = norm.gamma.double().cpu()
    d = 1e-5
    for i, j in ((0, 0), (1, 17), (2, 39)):
        dx = torch.zeros(rows, H, dtype=torch.float64)
        dx[i, j] = d
        want = (loss(x.double() + dx, gam) - loss(x.double() - dx, gam)) / (2 * d)      # differences: error d^2 |f'''| + 1e-16 |f| / d, both under 1e-8
        assert abs(float(xg.grad[i, j]) - want) < 1e-4 * max(1.0, abs(want))            # fp32 arithmetic on sums of 40 terms of order 1: 64 u * 40 < 2e-4 / 1.2
    for j in (0, 39):
        dg = torch.zeros(H, dtype=torch.float64)
        dg[j] = d
        want = (loss(x.double(), gam + dg) - loss(x.double(), gam - dg)) / (2 * d)
        assert abs(float(norm.ggamma[j]) - want) < 1e-4 * max(1.0, abs(want))
    assert torch.equal(xg.grad, rg.grad)
    # only the residual stream used: the addition's gradient alone
    norm.ggamma.zero_()
    xg.grad = rg.grad = None
    layers.rms_norm(xg, norm, residual=rg)[1].sum().backward()
    assert bool((xg.grad == 1).all()) and bool((rg.grad == 1).all()) and float(norm.ggamma.abs().sum()) == 0.0
    z = layers.rms_norm(xg, norm)
    xg.grad = None
    z.sum().backward()
    assert bool(torch.isfinite(xg.grad).all()) and float(norm.ggamma.abs().sum()) > 0.0
