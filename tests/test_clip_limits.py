"""CPU: the clip's limit on the elements of one call is the one it states, and is found before anything is launched (also where the tensors' table takes launches of its own)."""
import ctypes

import pytest

from merlot_amd import lib

P = 1 << 20                                                    # an address that is never touched: every call below is refused


def _clip(numels, types):
    n = len(numels)
    ins, ns = (ctypes.c_int64 * n)(*[P] * n), (ctypes.c_int64 * n)(*numels)
    d = lib.LIB.load()
    rc = d.merlot_clip_by_global_norm(ctypes.addressof(ins), None, ctypes.addressof(ns), ctypes.cast(bytes(types), ctypes.c_void_p), n, 0.0, P, P, 1 << 20, None)
    return rc, d.merlot_last_error().decode()


@pytest.mark.parametrize('kind', [0, 1])
@pytest.mark.parametrize('small', [0, 200])
def test_more_elements_than_the_limit(kind, small):
    big = (1 << 40) - 1
    rc, msg = _clip([1] * small + [big] * 8, [kind] * (small + 8))
    assert rc == -1 and '2^43 elements' in msg
    rc, msg = _clip([1] * small + [1 << 40], [kind] * (small + 1))
    assert rc < 0 and 'bad size' in msg

