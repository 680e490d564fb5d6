"""CPU: the entries of the norm, the 8-bit blocks and the clip refuse bad calls before any launch, and the test definitions hold against torch's own conversions."""
import ctypes

import pytest
import torch

import blocks_ref as ref
from merlot_amd import lib


def _call(name, *args):
    d = lib.LIB.load()
    return getattr(d, name)(*args), d.merlot_last_error().decode()


P = 4096                                                       # an address that is never touched: every call below is refused


def test_norm_refusals():
    ok = dict(x=P, ldx=768, f=0, res=None, ldr=0, gamma=P, h=None, y=P, rstd=P, y8=None, ld8=0, s8=None, lds8=0, rows=4, H=768, eps=1e-6, st=None)

    def fwd(**kw):
        return _call('merlot_rms_fwd', *{**ok, **kw}.values())
    for kw, what in ((dict(x=None), 'null operand'), (dict(gamma=None), 'null operand'), (dict(y=None), 'null operand'), (dict(rows=0), 'rows'), (dict(H=0), 'H=0'),
                     (dict(H=16385, ldx=20000), 'H=16385'), (dict(ldx=767), 'stride'), (dict(res=P, ldr=100, h=P), 'stride'), (dict(res=P, ldr=768), 'h is written'),
                     (dict(h=P), 'h is written'), (dict(y8=P, ld8=760, s8=P, lds8=8), '8-bit copy'), (dict(y8=P, ld8=768, s8=None, lds8=8), '8-bit copy'),
                     (dict(y8=P + 4, ld8=768, s8=P, lds8=8), 'aligned')):
        rc, msg = fwd(**kw)
        assert rc < 0 and what in msg, (kw, rc, msg)
    ok = dict(dy=P, lddy=768, f=0, h=P, ldh=768, rstd=P, gamma=P, dres=None, lddr=0, dx=P, dg=P, rows=4, H=768, ws=P, wsb=1 << 20, st=None)
    for kw, what in ((dict(dy=None), 'null'), (dict(dg=None), 'null'), (dict(rows=-1), 'rows'), (dict(H=20000, lddy=20000, ldh=20000), 'H=20000'), (dict(ldh=700), 'stride'),
                     (dict(dres=P, lddr=3), 'stride'), (dict(ws=None), 'workspace'), (dict(wsb=3071), 'workspace')):
        rc, msg = _call('merlot_rms_bwd', *{**ok, **kw}.values())
        assert rc < 0 and what in msg, (kw, rc, msg)
    q = lib.LIB.query
    assert q('merlot_rms_bwd_workspace_bytes', 4, 768) == 768 * 4 and q('merlot_rms_bwd_workspace_bytes', 0, 768) == 0 and q('merlot_rms_bwd_workspace_bytes', 4, 20000) == 0


def test_block_refusals():
    ok = dict(x=P, ldx=300, f=0, R=200, C=300, fmt=0, tile=1, q=P, ldq=384, s=P, lds=4, qt=P, ldqt=256, st=P, ldst=4, stream=None)
    for kw, what in ((dict(x=None), 'null'), (dict(q=None, qt=None), 'null'), (dict(s=None), 'null'), (dict(st=None), 'null'), (dict(R=0), 'empty'), (dict(C=0), 'empty'),
                     (dict(ldx=299), 'empty'), (dict(fmt=2), 'fmt'), (dict(tile=64), 'tile'), (dict(ldq=300), 'row-wise'), (dict(lds=2), 'row-wise'), (dict(ldqt=200), 'transposed'),
                     (dict(ldqt=260), 'transposed'), (dict(q=P + 8), 'aligned')):
        rc, msg = _call('merlot_quantize_blocks', *{**ok, **kw}.values())
        assert rc < 0 and what in msg, (kw, rc, msg)
    ok = dict(a=P, lda=256, fa=0, sa=P, lsa=4, b=P, ldb=256, sb=P, lsb=4, c=P, ldc=300, M=5000, N=300, K=256, f=0, acc=0, bias=None, ws=None, wsb=0, st=None)
    for kw, what in ((dict(a=None), 'null'), (dict(sb=None), 'null'), (dict(M=0), 'size'), (dict(N=0), 'size'), (dict(K=250), 'size'), (dict(K=0), 'size'), (dict(fa=2), 'fmt_a'),
                     (dict(acc=1), 'accumulation'), (dict(lda=128), 'leading'), (dict(ldc=299), 'leading'), (dict(lda=264), 'aligned'), (dict(b=P + 8), 'aligned'),
                     (dict(lsa=1), 'scale'), (dict(lsb=6), 'scale'), (dict(sa=P + 2), 'scale'), (dict(M=200, K=8192, lda=8192, ldb=8192, lsa=64, lsb=64), 'workspace')):
        rc, msg = _call('merlot_gemm_f8_blocks', *{**ok, **kw}.values())
        assert rc < 0 and what in msg, (kw, rc, msg)


def test_clip_refusals_and_overlaps():
    def clip(ins, outs, ns, types, c=1.0, norm=P, ws=P, wsb=1 << 20):
        n = len(ins)
        arr = lambda v: ctypes.addressof((ctypes.c_int64 * n)(*v)) if v is not None else None  # noqa: E731
        keep = [(ctypes.c_int64 * n)(*v) if v is not None else None for v in (ins, outs, ns)]
        a = [ctypes.addressof(k) if k is not None else None for k in keep]
        return _call('merlot_clip_by_global_norm', a[0], a[1], a[2], ctypes.cast(bytes(types), ctypes.c_void_p), n, c, norm, ws, wsb, None)
    cases = [(dict(ins=[], outs=[], ns=[], types=[]), 'no tensors'),
             (dict(ins=[P], outs=[P], ns=[4], types=[0], c=-1.0), 'clip must'), (dict(ins=[P], outs=[P], ns=[4], types=[0], c=float('nan')), 'clip must'),
             (dict(ins=[P], outs=[P], ns=[4], types=[0], c=float('inf')), 'clip must'), (dict(ins=[P], outs=None, ns=[4], types=[0]), 'null operand'),
             (dict(ins=[P], outs=[P], ns=[4], types=[0], ws=None), 'workspace'), (dict(ins=[P], outs=[P], ns=[4], types=[0], wsb=100), 'workspace'),
             (dict(ins=[P], outs=[P], ns=[-1], types=[0]), 'bad size'), (dict(ins=[P], outs=[P], ns=[4], types=[4]), 'bad type'), (dict(ins=[0], outs=[P], ns=[4], types=[0]), 'null tensor'),
             (dict(ins=[P + 2], outs=[P + 2], ns=[4], types=[0]), 'aligned'), (dict(ins=[P + 1], outs=[P + 1], ns=[4], types=[3]), 'aligned'),
             (dict(ins=[P, P], outs=[P, P], ns=[4, 4], types=[0, 0]), 'overlap'), (dict(ins=[P, P + 8], outs=[P, P + 8], ns=[4, 4], types=[0, 0]), 'overlap'),
             (dict(ins=[P, 8192], outs=[8192, P], ns=[4, 4], types=[0, 0]), 'overlap'), (dict(ins=[P], outs=[P + 4], ns=[4], types=[0]), 'overlap'),
             (dict(ins=[P], outs=[P], ns=[8], types=[1]), 'overlap'),           # in place with another type
             (dict(ins=[P, 20000, 8192], outs=[P, 30000, 40000], ns=[64, 4, 1], types=[0, 0, 0], c=1.0, ws=None), 'workspace'),
             (dict(ins=[P, P + 16, 8192], outs=[20480, 24576, P + 200], ns=[64, 2, 8], types=[0, 0, 0]), 'overlap')]   # a long input reaches past a short one that starts later
    for kw, what in cases:
        rc, msg = clip(**kw)
        assert rc < 0 and what in msg, (kw, rc, msg)
    q = lib.LIB.query
    assert q('merlot_clip_workspace_bytes', 1) == q('merlot_clip_workspace_bytes', 112) < q('merlot_clip_workspace_bytes', 113) and q('merlot_clip_workspace_bytes', 0) == 0


def test_python_refusals_need_no_device():
    from merlot_amd import ops
    for fn in (lambda: ops.rms_norm_fwd(torch.zeros(3, 4), torch.ones(4)), lambda: ops.quantize_blocks(torch.zeros(3, 4)), lambda: ops.clip_by_global_norm([torch.zeros(3)], 1.0),
               lambda: ops.global_norm([]), lambda: ops.rms_norm_fwd(torch.zeros(3, 4, dtype=torch.float16), torch.ones(4))):
        with pytest.raises(ValueError):
            fn()


@pytest.mark.parametrize('fmt', [0, 1])
def test_definition_of_the_blocks(fmt):
    """tests/blocks_ref.py against torch's own conversion to the format (nearest, ties to even) of exactly scaled values"""
    g = torch.Generator().manual_seed(fmt)
    x = (torch.randn(50, 300, generator=g) * torch.exp(4 * torch.randn(50, 1, generator=g))).bfloat16()
    q, s, v = ref.quantize(x, fmt)
    dt, top, mant, _ = ref.FORMATS[fmt]
    xp = torch.nn.functional.pad(x.double(), (0, 84)).view(50, 3, 128)
    two = ref.pow2(s.long() - 127).unsqueeze(-1)
    assert torch.equal((xp / two).float().to(dt).view(50, -1).view(torch.uint8), q.view(torch.uint8))
    amax = xp.abs().amax(-1, keepdim=True)
    assert bool((amax <= 1.75 * 2.0 ** top * two).all()) and bool((amax > 1.75 * 2.0 ** top * two / 2).all())
    assert torch.equal(ref.values(q, s), v)
