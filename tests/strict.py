"""TEST-ONLY comparison that nothing slips through: a NaN fails it (every comparison with a NaN is false, so 'no element is further off' would let it pass)."""


def close(got, want, tol, what):
    """every element of got within tol of want, both finite or not compared at all; the shapes are equal"""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, tuple(got.shape), tuple(want.shape))
    ok = (got - want).abs() <= tol
    assert bool(ok.all()), (what, int((~ok).sum()), 'of', ok.numel(), 'off; at', (~ok).nonzero()[0].tolist(), float(got[~ok][0]), float(want[~ok][0]))
