"""Global norm and clipping over many tensors (merlot_clip_by_global_norm, ops.global_norm / clip_by_global_norm) against 64 bits.

Tolerances: the norm is summed in 64 bits and rounded once (2^-24), the factor's division rounds once more, an fp32 output once more (3 * 2^-24 in all, 4 taken), a bf16 output to
half a step 2^-8."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _ops():
    from merlot_amd import ops
    return ops


def _tensors(sizes, kinds, seed, scale=1.0, shift=0):
    """tensors of the given sizes, `shift` elements into an allocation of their own (alignment)"""
    g = torch.Generator().manual_seed(seed)
    host = [(torch.randn(n, generator=g) * scale).to(k) for n, k in zip(sizes, kinds)]
    dev = []
    for i, t in enumerate(host):
        base = torch.full((t.numel() + 16,), 7.0, device='cuda', dtype=t.dtype)
        s = (shift * (i + 1)) % 9
        base[s:s + t.numel()] = t.cuda()
        dev.append((base, s))
    return host, [b[s:s + t.numel()] for (b, s), t in zip(dev, host)], dev


def _check(host, got, norm, clip, out_kinds):
    n64 = sum(float(t.double().pow(2).sum()) for t in host) ** 0.5
    assert abs(float(norm) - n64) <= 2 * U * n64
    f = clip / max(n64, clip)
    for t, o, k in zip(host, got, out_kinds):
        want = t.double() * f
        tol = want.abs() * ((2.0 ** -8 if k == torch.bfloat16 else 0.0) + 4 * U) + 1e-40
        assert bool(((o.double().cpu() - want).abs() <= tol).all()), (t.numel(), t.dtype, k)


F, B = torch.float32, torch.bfloat16


@pytest.mark.parametrize('shift', [0, 1, 3])
@pytest.mark.parametrize('clip', [1.0, 1e6])
@pytest.mark.parametrize('sizes', [[1], [0, 5], [3, 1, 4, 15, 9, 2], [8191, 8192, 8193, 16385], [100003, 7, 50000], list(range(1, 400, 3))])
def test_mixed_tensors(sizes, clip, shift):
    ops = _ops()
    kinds = [B if i % 3 == 1 else F for i in range(len(sizes))]
    host, dev, base = _tensors(sizes, kinds, len(sizes) + shift, 0.3, shift)
    assert abs(float(ops.global_norm(dev)) - sum(float(t.double().pow(2).sum()) for t in host) ** 0.5) <= 2 * U * max(1.0, float(ops.global_norm(dev)))
    outs = [torch.empty(n, device='cuda', dtype=B if i % 4 == 2 else F) for i, n in enumerate(sizes)]
    norm = ops.clip_by_global_norm(dev, clip, out=outs)
    _check(host, outs, norm, clip, [o.dtype for o in outs])
    for t, d in zip(host, dev):
        assert torch.equal(d.cpu(), t)                         # the inputs stay
    norm = ops.clip_by_global_norm(dev, clip)
    _check(host, dev, norm, clip, kinds)
    for (b, s), t in zip(base, host):                          # nothing outside the tensors is written
        assert bool((b[:s] == 7).all()) and bool((b[s + t.numel():] == 7).all())
    if clip == 1e6:
        assert all(torch.equal(d.cpu(), t) for t, d in zip(host, dev))


@pytest.mark.parametrize('into', [F, B])
@pytest.mark.parametrize('kind', [F, B])
def test_outputs_at_any_offset(kind, into):
    """inputs and outputs that start at different places of their 16 bytes; nothing beside the outputs is written"""
    ops = _ops()
    sizes = [9, 4096, 5001, 12289, 700, 33, 8192, 20000, 15]
    host, dev, _ = _tensors(sizes, [kind] * len(sizes), 3, 0.1, 1)
    bases = [torch.full((n + 32,), 7.0, device='cuda', dtype=into) for n in sizes]
    for first in (0, 1, 2, 5):
        outs = [b[(first + 3 * i) % 8:][:n] for i, (b, n) in enumerate(zip(bases, sizes))]
        _check(host, outs, ops.clip_by_global_norm(dev, 2.0, out=outs), 2.0, [into] * len(sizes))
        for i, (b, n) in enumerate(zip(bases, sizes)):
            s = (first + 3 * i) % 8
            assert bool((b[:s] == 7).all()) and bool((b[s + n:] == 7).all())
            b.fill_(7.0)


def test_more_tensors_than_one_launch_takes_and_a_kept_list():
    ops = _ops()
    sizes = [1 + (i * 37) % 1500 for i in range(300)]
    kinds = [F] * 300
    host, dev, _ = _tensors(sizes, kinds, 9, 0.01)
    kept, flat = ops.TensorList(dev), torch.empty(sum(sizes), device='cuda')
    outs = ops.TensorList(flat.split(sizes))
    first = None
    for _ in range(3):
        flat.zero_()
        norm = ops.clip_by_global_norm(kept, 0.25, out=outs)
        _check(host, outs.tensors, norm, 0.25, kinds)
        first = flat.clone() if first is None else first
        assert torch.equal(first, flat)                        # a fixed order of sums: the same bits
    for t in dev:
        t.mul_(2.0)                                            # new values behind a kept list
    _check([2 * t for t in host], outs.tensors, ops.clip_by_global_norm(kept, 0.25, out=outs), 0.25, kinds)


def test_norms_that_are_not_finite_and_large_values():
    ops = _ops()
    a, b = torch.full((1000,), 3e30, device='cuda'), torch.ones(10, device='cuda')
    assert abs(float(ops.global_norm([a, b])) - 3e30 * 1000 ** 0.5) < 1e24 * 30          # squares of 9e60: no overflow in 64 bits
    t = torch.tensor([1.0, float('inf'), -2.0], device='cuda')
    assert float(ops.clip_by_global_norm([t, b], 1.0)) == float('inf')
    assert float(t[0]) == 0.0 and bool(torch.isnan(t[1])) and bool((b == 0).all())
    t, b = torch.tensor([1.0, float('nan')], device='cuda'), torch.ones(10, device='cuda', dtype=B)
    assert bool(torch.isnan(ops.clip_by_global_norm([t, b], 1.0)))
    assert bool(torch.isnan(t).all()) and bool(torch.isnan(b).all())
    z = torch.zeros(5, device='cuda')
    assert float(ops.clip_by_global_norm([z], 1.0)) == 0.0 and bool((z == 0).all())


def test_optimizer_clips_through_the_kernel():
    """AdamOptimizer.clip_local_gradients on a device arena: the rule of tf.clip_by_global_norm over everything that is not frozen"""
    from common import tiny_config
    from merlot_amd import ParamStore
    from merlot_amd.optimization import AdamOptimizer
    st = ParamStore(tiny_config(), 'cuda:0', seed=0)
    opt = AdamOptimizer(st, 1e-3, 100, 10, freeze_scope='contrastive', clip_norm=0.5)
    g = torch.Generator().manual_seed(1)
    st.grad.copy_(torch.randn(st.grad.shape, generator=g) * 1e-2)
    for name, (off, n, _) in st.offsets.items():
        st.grad[off + n:off + (n + 63) // 64 * 64] = 0
    ref = st.grad.double().cpu()
    for s, e in opt.frozen:
        ref[s:e] = 0
    norm = opt.clip_local_gradients()
    want = float(ref.norm())
    assert norm.shape == () and abs(float(norm) - want) <= 2 * U * want
    assert bool(((st.grad.double().cpu() - ref * (0.5 / want)).abs() <= ref.abs() * (0.5 / want) * 4 * U).all())
    opt.clip_norm = 0.0
    before = st.grad.clone()
    assert abs(float(opt.clip_local_gradients()) - 0.5) < 1e-6 and torch.equal(before, st.grad)


def test_refusals_on_the_device():
    ops = _ops()
    a, b = torch.ones(64, device='cuda'), torch.ones(64, device='cuda')
    for bad in ([a, a], [a, a[32:]], [a[:40], a[32:]]):
        with pytest.raises(Exception, match='overlap'):
            ops.clip_by_global_norm(bad, 1.0)
    with pytest.raises(Exception, match='overlap'):
        ops.clip_by_global_norm([a, b], 1.0, out=[b, a])           # exchanged in place: an element would be read after it was written
    with pytest.raises(Exception, match='overlap'):
        ops.clip_by_global_norm([a.view(torch.bfloat16)[:64]], 1.0, out=[a])
    for bad, what in (([], 'no tensors'), ([torch.ones(3)], 'GPU tensor'), ([a.half()], 'f32 or bf16'), ([torch.ones(4, 4, device='cuda').t()], 'contiguous')):
        with pytest.raises(ValueError, match=what):
            ops.clip_by_global_norm(bad, 1.0)
    for clip in (0.0, -1.0, float('inf'), float('nan')):
        with pytest.raises(ValueError, match='clip_norm'):
            ops.clip_by_global_norm([a], clip)
    with pytest.raises(ValueError, match='same shapes'):
        ops.clip_by_global_norm([a], 1.0, out=[b[:32]])
    kept = ops.TensorList([a, b])
    b.data = torch.ones(64, device='cuda')
    with pytest.raises(ValueError, match='has changed'):
        ops.global_norm(kept)
    assert bool((a == 1).all())
    # the norm alone may count a tensor twice; sqrt(128) is no fp32 number: half a step off at most
    assert abs(float(ops.global_norm([a, a])) - 128 ** 0.5) <= U * 128 ** 0.5
