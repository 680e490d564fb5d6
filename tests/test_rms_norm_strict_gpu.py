"""The root-mean-square norm's numeric tests with a comparison that a NaN fails (tests/strict.py): an output that nothing wrote, or a row's bad statistics, show as NaN."""
import pytest
import torch

import strict
import test_rms_norm_gpu as base

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _strict(monkeypatch):
    monkeypatch.setattr(base, '_close', strict.close)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('H', base.WIDTHS)
def test_forward_and_backward(H, dtype):
    base.test_forward_and_backward(H, dtype)


def test_many_rows():
    base.test_many_rows_take_every_loop_iteration()


def test_extremes():
    base.test_zeros_extremes_and_rows_that_are_not_finite()
