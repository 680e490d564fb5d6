"""CPU: the comparison of tests/strict.py rejects what it has to."""
import pytest
import torch

import strict


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf'), 1.3])
def test_one_bad_element_fails(bad):
    want = torch.ones(3, 5, dtype=torch.float64)
    tol = torch.full((3, 5), 0.25, dtype=torch.float64)
    got = torch.full((3, 5), 1.25)
    strict.close(got, want, tol, 'at the border')
    got[2, 4] = bad
    with pytest.raises(AssertionError, match='1, .of., 15'):
        strict.close(got, want, tol, 'y')


def test_shapes_and_nan_in_the_reference_fail():
    want = torch.ones(3, dtype=torch.float64)
    with pytest.raises(AssertionError):
        strict.close(torch.ones(1), want, torch.ones(3), 'broadcast')
    with pytest.raises(AssertionError):
        strict.close(torch.ones(3), want * float('nan'), torch.ones(3), 'reference')
    with pytest.raises(AssertionError):
        strict.close(torch.ones(3), want, torch.full((3,), float('nan')), 'tolerance')
