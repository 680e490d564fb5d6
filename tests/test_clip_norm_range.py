"""CPU: a clip_norm that fp32 cannot hold is refused, not taken as 0 (which asks for the norm alone and leaves every output as it was) or as infinite."""
import pytest
import torch

from merlot_amd import ops


@pytest.mark.parametrize('clip', [1e-50, 5e-324, 2.0 ** -150, 1e39, 3.5e38, float('inf'), float('nan'), 0.0, -1.0, -1e-50])
def test_refused(clip):
    with pytest.raises(ValueError, match='clip_norm'):
        ops.clip_by_global_norm([torch.zeros(3)], clip)


@pytest.mark.parametrize('clip', [1e-45, 1.2e-38, 1, 3.4e38])
def test_accepted(clip):
    with pytest.raises(ValueError, match='GPU tensor'):       # the next check: the tensors are not the device's
        ops.clip_by_global_norm([torch.zeros(3)], clip)
