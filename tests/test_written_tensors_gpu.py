"""What the norm, the 8-bit product and the clip write in place counts as written: autograd refuses a backward over a tensor that was saved before, and gives no
gradient of values that are gone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _saved(t):
    """a graph that has saved t"""
    w = torch.ones_like(t, requires_grad=True)
    return (w * t).sum()


def _stale(loss):
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_clipping_in_place_and_into_outputs():
    from merlot_amd import ops
    a, b = torch.ones(100, device='cuda'), torch.ones(50, device='cuda', dtype=torch.bfloat16)
    arena = torch.zeros(200, device='cuda')
    outs = [arena[:100], arena[100:150]]
    la, lb, lo = _saved(a), _saved(b), _saved(arena)
    ops.clip_by_global_norm([a, b], 1.0, out=outs)
    _stale(lo)                                                 # (a view's write is its base's)
    la.backward(retain_graph=True)                             # the inputs were read only
    ops.clip_by_global_norm([a, b], 1.0)
    _stale(la)
    _stale(lb)
    before = a._version
    ops.global_norm([a])
    assert a._version == before
    kept = ops.TensorList([a])
    l2 = _saved(a)
    ops.clip_by_global_norm(kept, 0.5)
    _stale(l2)


def test_the_norms_gain_gradient_and_the_products_output():
    from merlot_amd import ops
    x, gamma, dg = torch.randn(8, 64, device='cuda'), torch.ones(64, device='cuda'), torch.zeros(64, device='cuda')
    _, _, rstd, _, _ = ops.rms_norm_fwd(x, gamma)
    loss, same = _saved(dg), _saved(x)
    ops.rms_norm_bwd(x, x, rstd, gamma, dg)
    _stale(loss)
    same.backward()
    q, s = ops.quantize_blocks(torch.randn(16, 128, device='cuda'))
    out = torch.zeros(16, 16, device='cuda')
    loss = _saved(out)
    ops.gemm_f8_blocks(q, s, q, s, out=out)
    _stale(loss)
    loss = _saved(out)
    ops.gemm_f8_blocks(q, s, q, s, out=out, accumulate=True)
    _stale(loss)


def test_inference_tensors_have_no_version():
    from merlot_amd import ops
    with torch.inference_mode():
        a = torch.ones(100, device='cuda')
        assert abs(float(ops.clip_by_global_norm([a], 1.0)) - 10.0) < 1e-5
    assert bool((a.clone() - 0.1).abs().max() < 1e-7)
    ops.clip_by_global_norm([a], 0.5)
