"""CPU: rows and row strides as ops._rows takes them from a tensor's layout (the device is the CPU's own -1 here)."""
import pytest
import torch

from merlot_amd import ops


def _rows(t):
    return ops._rows(t, t.dtype, -1, 't')


def test_layouts():
    x = torch.zeros(6, 8)
    assert _rows(x) == (6, 8, 8) and _rows(x[:, 2:5]) == (6, 3, 8) and _rows(x[2:3, :5]) == (1, 5, 5) and _rows(x[0]) == (1, 8, 8)
    assert _rows(torch.zeros(2, 3, 8)) == (6, 8, 8) and _rows(torch.zeros(2, 3, 8)[..., :4]) == (6, 4, 8) and _rows(torch.zeros(0, 8)) == (0, 8, 8)
    for bad in (x.t(), x[:, ::2], x[:1].expand(6, 8), torch.zeros(3, 2, 8).transpose(0, 1), torch.zeros(())):
        with pytest.raises(ValueError):
            _rows(bad)


def test_the_stride_of_a_single_column_does_not_matter():
    """[N, 1] is contiguous whatever the stride of its one column, and torch leaves any there"""
    x = torch.zeros(1, 6).t()
    assert x.is_contiguous() and x.stride() == (1, 6)
    assert _rows(x) == (6, 1, 1)
    assert _rows(torch.zeros(4, 6).as_strided((6, 1), (4, 3))) == (6, 1, 4)
    assert _rows(torch.zeros(1, 2, 3).permute(1, 2, 0)) == (6, 1, 1)
    s = torch.zeros(24, dtype=torch.uint8)
    assert ops._scale_rows(s.as_strided((6, 1), (4, 9)), 6, 1, -1, 's') == 4
    with pytest.raises(ValueError, match='overlap'):
        _rows(torch.zeros(6).as_strided((6, 1), (0, 1)))
