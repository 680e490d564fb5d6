"""ops.TensorList: a kept list notices every way in which one of its tensors can come to mean other elements than the list was made for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _resize(t):
    t.resize_(32)


def _shorter(t):
    t.data = t.data[:32]


def _longer(t):
    t.data = t.data.as_strided((96,), (1,))


def _apart(t):
    t.data = t.data.as_strided((64,), (2,))


def _elsewhere(t):
    t.data = torch.ones(64, device='cuda')



@pytest.mark.parametrize('change', [_resize, _shorter, _longer, _apart, _elsewhere])
def test_a_changed_tensor_is_refused(change):
    from merlot_amd import ops
    base = torch.ones(128, device='cuda')
    a, b = torch.ones(64, device='cuda'), base[:64].detach()
    kept, other = ops.TensorList([a, b]), ops.TensorList([torch.zeros(64, device='cuda') for _ in range(2)])
    assert float(ops.global_norm(kept)) ** 2 == pytest.approx(128, rel=1e-6)
    change(b)
    for call in (lambda: ops.global_norm(kept), lambda: ops.clip_by_global_norm(kept, 0.5), lambda: ops.clip_by_global_norm(kept, 0.5, out=other),
                 lambda: ops.clip_by_global_norm(other, 0.5, out=kept)):
        with pytest.raises(ValueError, match='has changed'):
            call()
    assert bool((base == 1).all()) and bool((a == 1).all())


def test_other_shapes_of_the_same_elements_are_none():
    from merlot_amd import ops
    a = torch.ones(64, device='cuda')
    kept = ops.TensorList([a])
    a.data = a.data.view(8, 8)
    assert abs(float(ops.clip_by_global_norm(kept, 1.0)) - 8.0) < 1e-6 and bool((a == 0.125).all())
