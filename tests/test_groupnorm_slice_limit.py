"""CPU: the one-launch GroupNorm entries wait inside the kernel and stop returning above a number of slices per sample; the limit that keeps them under it is a constant
that no environment variable and no build lifts, and no script looks for the place where it breaks."""
import os

import pytest

from merlot_amd import lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096                                                       # an address that is never touched: every call below is refused


@pytest.mark.parametrize('name', ['MERLOT_GN_MAX_SLICES', 'MERLOT_GN_STATIC'])
def test_more_slices_are_refused_whatever_the_environment(monkeypatch, name):
    monkeypatch.setenv(name, '100000')
    d = lib.LIB.load()
    N, W, C, G = 1, 64, 64, 32
    for H in (165, 4000):                                      # 256 positions per slice backward (41.25: 42 slices), 512 forward
        rc = d.merlot_groupnorm_bwd_fused(P, None, P, P, P, P, P, P, P, P, None, N, H, W, C, G, 1e-4, 1, P, 1 << 40, None)
        assert rc < 0 and 'slices per sample' in d.merlot_last_error().decode(), H
    rc = d.merlot_groupnorm_fwd_fused(P, P, P, None, P, P, N, 330, W, C, G, 1e-4, 1, P, 1 << 40, None)
    assert rc < 0 and 'slices per sample' in d.merlot_last_error().decode()
    assert ops.GN_FUSED_MAX_SLICES == 40


def test_no_source_or_script_lifts_the_limit():
    for folder in ('merlot_amd/csrc', 'scripts'):
        for f in sorted(os.listdir(os.path.join(ROOT, folder))):
            if f.endswith(('.hip', '.inc', '.h', '.py', '.sh')):
                text = open(os.path.join(ROOT, folder, f)).read()
                assert 'GN_MAX_SLICES' not in text.replace('GN_FUSED_MAX_SLICES', '') and 'GN_STATIC' not in text and 'GN_FUSED_MAX_SLICES = 1' not in text, f
