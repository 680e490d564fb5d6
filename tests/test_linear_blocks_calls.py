"""CPU: what layers.linear_f8_blocks asks of the 8-bit operators, with those operators replaced by ones that take notes."""
import pytest
import torch

from merlot_amd import layers, ops


class _Lin(object):
    def __init__(self, n, k, bias):
        self.w = torch.zeros(n, k)
        self.wb, self.gw = self.w.bfloat16(), torch.zeros(n, k)
        self.b = self.gb = torch.zeros(n) if bias else None


@pytest.fixture
def notes(monkeypatch):
    made = []

    def quantize(x, fmt=0, *, tile=1, rows=True, transpose=False):
        made.append(transpose)
        q, s = x.new_empty(x.shape), x.new_empty(1)
        return (q, s, q.t().clone(), s.clone()) if transpose else (q, s)
    monkeypatch.setattr(ops, 'quantize_blocks', quantize)
    monkeypatch.setattr(ops, 'gemm_f8_blocks', lambda a, sa, b, sb, **kw: torch.zeros(a.shape[0], b.shape[0], dtype=torch.bfloat16))
    return made


def test_transposed_copies_only_where_a_backward_may_follow(notes):
    lin = _Lin(8, 16, False)
    x = torch.zeros(4, 16, requires_grad=True)
    y = layers.linear_f8_blocks(x, lin)
    assert y.requires_grad and notes == [True, True]
    for call in (lambda: layers.linear_f8_blocks(x.detach(), lin), lambda: torch.no_grad()(layers.linear_f8_blocks)(x, lin)):
        del notes[:]
        y = call()
        assert not y.requires_grad and y.shape == (4, 8) and notes == [False, False]


def test_any_output_width_without_a_backward(notes):
    lin = _Lin(6, 16, True)
    x = torch.zeros(4, 16, requires_grad=True)
    with pytest.raises(ValueError, match='multiple of 4'):     # the bias gradient's column sums
        layers.linear_f8_blocks(x, lin)
    assert notes == []
    with torch.no_grad():
        assert layers.linear_f8_blocks(x, lin).shape == (4, 6)
    assert layers.linear_f8_blocks(x.detach(), lin).shape == (4, 6)


@pytest.mark.parametrize('rows', [(1 << 22) - 127, 1 << 22])
def test_more_rows_than_the_weight_gradient_takes_are_refused_in_the_forward(notes, rows):
    """(the product of the backward, whose reduction they are, refuses them: too late, the step's other gradients are on their way)"""
    lin = _Lin(8, 1, False)
    x = torch.zeros(rows, 1, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match='4194176'):
        layers.linear_f8_blocks(x, lin)
    assert notes == []
    assert layers.linear_f8_blocks(x.detach(), lin).shape == (rows, 8)
    assert layers.linear_f8_blocks(x[:ops.F8_BLOCKS_MAX_K], lin).requires_grad
    d = ops.LIB.load()
    P, K = 4096, ops.F8_BLOCKS_MAX_K                           # the product's own limit (refused before any launch)
    call = lambda k, ws: (d.merlot_gemm_f8_blocks(P, k, 0, P, 1 << 15, P, k, P, 1 << 15, P, 8, 8, 8, k, 1, 0, None, None, ws, None), d.merlot_last_error().decode())  # noqa: E731
    assert 'leading dimension' in call(K + 128, 0)[1] and 'workspace' in call(K, 0)[1]
