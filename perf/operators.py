"""The operators of a training step on 8-bit blocks, their inputs and what they cost.

Four kinds of case:
  norm     root-mean-square norm of x (+ a residual), forward alone or forward and backward
  chain    the same norm with its output in 8 bits, a scale for each 128 features, and the 8-bit product that reads it
  product  the product of two 8-bit operands with a scale for each block of 128 along the reduction
  linear   one Linear of a training step on such operands, from bf16: output, input gradient and weight gradient
  clip     the global norm of many gradients, and the gradients scaled by clip / max(norm, clip)

An 8-bit operand [R, K] has its columns padded with zeros to whole blocks of 128; its scales are bytes [R, K / 128] (row stride a multiple of 4) and a
byte b stands for 2^(b - 127), the smallest power of two that brings the block's largest magnitude under the format's largest value.
"""
import math

import torch

own = False

EPS = 1e-6
TOP = {'e4m3': (torch.float8_e4m3fn, 8), 'e5m2': (torch.float8_e5m2, 15)}      # largest value = 1.75 * 2^exponent
DTYPES = {'bf16': torch.bfloat16, 'f32': torch.float32}


def listed():
    return [
        # one new token through a block's first norm and its fused Q | K | V product (hidden size 768): latency
        {'name': 'chain, one token', 'op': 'chain', 'rows': 1, 'H': 768, 'N': 2304, 'pad': 0},
        # the captions of a batch of videos through a norm and a square product
        {'name': 'chain, captions', 'op': 'chain', 'rows': 65536, 'H': 768, 'N': 768, 'pad': 0},
        # the norm of one row alone: the smallest call
        {'name': 'norm, one row', 'op': 'norm', 'rows': 1, 'H': 1024, 'dtype': 'bf16', 'residual': True, 'backward': False, 'pad': 0},
        # a norm of the frames' patch tokens in training
        {'name': 'norm step, patches', 'op': 'norm', 'rows': 101376, 'H': 768, 'dtype': 'bf16', 'residual': True, 'backward': True, 'pad': 0},
        # a head's norm in 32 bits, on a view of a wider buffer, odd sizes
        {'name': 'norm step, odd head', 'op': 'norm', 'rows': 4099, 'H': 1001, 'dtype': 'f32', 'residual': False, 'backward': True, 'pad': 7},
        # a few dozen tokens against a large weight: its bytes are what it costs
        {'name': 'product, 32 tokens', 'op': 'product', 'M': 32, 'N': 4096, 'K': 4096, 'fa': 'e4m3', 'fb': 'e4m3', 'out': 'bf16', 'bias': True},
        # the patch tokens' fused Q | K | V product
        {'name': 'product, qkv', 'op': 'product', 'M': 101376, 'N': 2304, 'K': 768, 'fa': 'e4m3', 'fb': 'e4m3', 'out': 'bf16', 'bias': True},
        # logits of masked positions over the whole vocabulary, a ragged number of them, a gradient's format on one side
        {'name': 'product, vocabulary', 'op': 'product', 'M': 4099, 'N': 50370, 'K': 768, 'fa': 'e5m2', 'fb': 'e4m3', 'out': 'f32', 'bias': True},
        # an MLP's first Linear in a training step
        {'name': 'linear step', 'op': 'linear', 'M': 32768, 'N': 4096, 'K': 1024, 'grad': 'e4m3'},
        # a head's Linear over a ragged number of rows
        {'name': 'linear step, ragged', 'op': 'linear', 'M': 700, 'N': 500, 'K': 1000, 'grad': 'e5m2'},
        # the gradients of a model held tensor by tensor: matrices, biases, gains
        {'name': 'clip, many tensors', 'op': 'clip', 'tensors': 300, 'largest': 1 << 21, 'total': 60_000_000, 'mixed': True, 'clip': 1.0, 'scale': 1e-3},
        # the gradients of this repository's model in one buffer
        {'name': 'clip, one buffer', 'op': 'clip', 'tensors': 1, 'largest': 223_000_001, 'total': 223_000_001, 'mixed': False, 'clip': 1.0, 'scale': 1e-3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['norm', 'chain', 'product', 'product', 'linear', 'clip'])
    if op == 'norm':
        H = _log(rng, 8, 8192)
        return {'op': op, 'rows': _log(rng, 1, max(1, min(101376, 75_000_000 // H))), 'H': H, 'dtype': rng.choice(['bf16', 'f32']), 'residual': rng.random() < 0.6,
                'backward': rng.random() < 0.6, 'pad': rng.choice([0, 0, 8, 3])}
    if op == 'chain':
        H = _log(rng, 32, 4096)
        N = _log(rng, 16, 4096)
        return {'op': op, 'rows': _log(rng, 1, max(1, min(65536, 50_000_000 // max(H, N)))), 'H': H, 'N': N, 'pad': rng.choice([0, 0, 8, 5])}
    if op == 'product':
        K = _log(rng, 16, 8192)
        N = _log(rng, 1, 50370)
        M = _log(rng, 1, max(1, min(101376, 200_000_000 // N, 75_000_000 // K, 150_000_000_000 // (N * K))))
        return {'op': op, 'M': M, 'N': N, 'K': K, 'fa': rng.choice(['e4m3', 'e4m3', 'e5m2']), 'fb': 'e4m3', 'out': rng.choice(['bf16', 'bf16', 'f32']),
                'bias': rng.random() < 0.5}
    if op == 'linear':
        K, N = _log(rng, 16, 4096), _log(rng, 16, 4096)
        return {'op': op, 'M': _log(rng, 1, max(1, min(32768, 130_000_000_000 // (N * K)))), 'N': N, 'K': K, 'grad': rng.choice(['e4m3', 'e5m2'])}
    n = _log(rng, 1, 400)
    return {'op': 'clip', 'tensors': n, 'largest': 1 << 22, 'total': _log(rng, n * 8, min(220_000_000, n << 22)), 'mixed': rng.random() < 0.5,
            'clip': rng.choice([1.0, 0.5, 100.0]), 'scale': rng.choice([1e-3, 1e-2])}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _pad128(n):
    return (n + 127) // 128 * 128


def _exponents(amax, top):
    """e of the smallest 2^e with amax <= 1.75 * 2^(top + e); 0 where there is nothing but zeros"""
    m, p = torch.frexp(amax)                                   # amax = m * 2^p, m in [0.5, 1)
    e = (p - 1 - top + (m > 0.875).to(p.dtype)).clamp(-127, 127)
    return torch.where(amax == 0, torch.zeros_like(e), e)


def _two(e):
    """2^e in 32 bits, exactly (a power function's last bit would decide ties), e in [-127, 127]"""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _blocks(x, fmt, tile=1):
    """x [R, C] in 32 bits -> the values its 8-bit copy stands for, [R, padded C] in 32 bits, their codes, and the exponents [R, blocks]"""
    dtype, top = TOP[fmt]
    R, C = x.shape
    x = torch.nn.functional.pad(x, (0, _pad128(C) - C)).contiguous()
    b = x.view(R, -1, 128)
    amax = b.abs().amax(-1)
    if tile > 1:
        up = torch.nn.functional.pad(amax, (0, 0, 0, _pad128(R) - R)).view(-1, 128, amax.shape[1]).amax(1)
        amax = up.repeat_interleave(128, 0)[:R]
    e = _exponents(amax, top)
    codes = (b * _two(-e).unsqueeze(-1)).to(dtype)
    return (codes.float() * _two(e).unsqueeze(-1)).view(R, -1), codes.view(R, -1), e


def _operand(x, fmt, tile=1):
    """the 8-bit copy of x as a program holds it: codes [R, K], scale bytes [R, K / 128] with a row stride that is a multiple of 4"""
    _, codes, e = _blocks(x, fmt, tile)
    s = torch.full((x.shape[0], (e.shape[1] + 3) // 4 * 4), 127, device=x.device, dtype=torch.uint8)
    s = s[:, :e.shape[1]]
    s.copy_((e + 127).to(torch.uint8))
    return codes, s


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device='cuda')


def _activations(g, rows, H, pad=0):
    """rows of different magnitude with a few features that stick out, as a residual stream has them"""
    x = _rand(g, rows, H + pad)
    x *= torch.exp(0.5 * _rand(g, rows, 1))
    x *= torch.where(torch.rand(H + pad, generator=g, device='cuda') < 0.01, 20.0, 1.0)
    return x


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    s = dict(case)
    if case['op'] in ('norm', 'chain'):
        rows, H, pad = case['rows'], case['H'], case['pad']
        dt = DTYPES[case.get('dtype', 'bf16')]
        s['x'] = _activations(g, rows, H, pad).to(dt)[:, :H]
        if case.get('residual', True):
            s['res'] = _activations(g, rows, H).to(dt)
        s['gamma'] = 1.0 + 0.1 * _rand(g, H)
        if case['op'] == 'chain':
            s['w'], s['sw'] = _operand(0.03 * _rand(g, case['N'], H), 'e4m3', 128)
        elif case['backward']:
            s['dy'] = (1e-3 * _rand(g, rows, H)).to(dt)
            s['dh'] = (1e-3 * _rand(g, rows, H)).to(dt)
    elif case['op'] == 'product':
        s['a'], s['sa'] = _operand(_activations(g, case['M'], case['K']), case['fa'])
        s['b'], s['sb'] = _operand(0.03 * _rand(g, case['N'], case['K']), case['fb'], 128)
        s['bias'] = 0.1 * _rand(g, case['N']) if case['bias'] else None
    elif case['op'] == 'linear':
        s['x'] = _activations(g, case['M'], case['K']).bfloat16()
        s['w'] = (0.03 * _rand(g, case['N'], case['K'])).bfloat16()
        s['dy'] = (1e-4 * _activations(g, case['M'], case['N'])).bfloat16()
    else:
        sizes = _sizes(case)
        kinds = [torch.bfloat16 if case['mixed'] and i % 4 == 1 else torch.float32 for i in range(len(sizes))]
        s['grads'] = [(case['scale'] * _rand(g, n)).to(k) for n, k in zip(sizes, kinds)]
        s['flat'] = torch.zeros(sum(sizes), device='cuda')
        s['outs'] = list(s['flat'].split(sizes))
        if own:                                                # the handle a program keeps for as long as its gradients stay where they are
            from merlot_amd import ops
            s['list'], s['out_list'] = ops.TensorList(s['grads']), ops.TensorList(s['outs'])
    return s


def _sizes(case):
    """the sizes of a clip's tensors: spread over their logarithm, `total` elements in all"""
    n, total = case['tensors'], case['total']
    if n == 1:
        return [min(total, case['largest'])]
    raw = [math.exp(((i * 7919) % n) / (n - 1) * math.log(4096.0)) for i in range(n)]
    k = total / sum(raw)
    return [max(1, min(case['largest'], int(r * k))) for r in raw]


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(state):
    return {'norm': _run_norm, 'chain': _run_chain, 'product': _run_product, 'linear': _run_linear, 'clip': _run_clip}[state['op']](state)


def _norm(x, res, gamma):
    """-> (h as stored, h in 32 bits, 1 / rms, y in 32 bits)"""
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.square().mean(-1, keepdim=True) + EPS)
    return h, hf, rstd, hf * rstd * gamma


def _run_norm(s):
    x, res, gamma = s['x'], s.get('res'), s['gamma']
    out = {}
    if own:
        from merlot_amd import ops
        y, h, rstd, _, _ = ops.rms_norm_fwd(x, gamma, residual=res, eps=EPS, save_rstd=s['backward'])
        if s['backward']:
            dgamma = torch.zeros_like(gamma)
            out['dx'] = ops.rms_norm_bwd(s['dy'], h if res is not None else x, rstd, gamma, dgamma, dres=s['dh'])
            out['dgamma'] = dgamma
    else:
        h, hf, rstd, y = _norm(x, res, gamma)
        y = y.to(x.dtype)
        if s['backward']:
            dy = s['dy'].float()
            t = dy * hf * rstd
            out['dx'] = (rstd * (dy * gamma - hf * rstd * (t * gamma).mean(-1, keepdim=True)) + s['dh'].float()).to(x.dtype)
            out['dgamma'] = t.sum(0)
    out['y'] = y
    if res is not None:
        out['h'] = h
    return out


def _values(q, s):
    """the values an 8-bit operand stands for, in 32 bits"""
    return (q.float().view(q.shape[0], -1, 128) * _two(s.int() - 127).unsqueeze(-1)).view(q.shape)


def _run_chain(s):
    if own:
        from merlot_amd import ops
        _, h, _, y8, s8 = ops.rms_norm_fwd(s['x'], s['gamma'], residual=s['res'], eps=EPS, save_rstd=False, out=False, q8=True)
        return {'h': h, 'out': ops.gemm_f8_blocks(y8, s8, s['w'], s['sw'])}
    h, _, _, y = _norm(s['x'], s['res'], s['gamma'])
    return {'h': h, 'out': (_blocks(y, 'e4m3')[0] @ _values(s['w'], s['sw']).T).bfloat16()}


def _run_product(s):
    if own:
        from merlot_amd import ops
        return ops.gemm_f8_blocks(s['a'], s['sa'], s['b'], s['sb'], bias=s['bias'], out_dtype=DTYPES[s['out']])
    c = _values(s['a'], s['sa']) @ _values(s['b'], s['sb']).T
    return (c if s['bias'] is None else c + s['bias']).to(DTYPES[s['out']])


def _run_linear(s):
    x, w, dy = s['x'], s['w'], s['dy']
    if own:
        from merlot_amd import ops
        fmt = ops.F8_E4M3 if s['grad'] == 'e4m3' else ops.F8_E5M2
        x8, sx, xt8, sxt = ops.quantize_blocks(x, transpose=True)
        w8, sw, wt8, swt = ops.quantize_blocks(w, tile=128, transpose=True)
        y = ops.gemm_f8_blocks(x8, sx, w8, sw)
        d8, sd, dt8, sdt = ops.quantize_blocks(dy, fmt, transpose=True)
        dx = ops.gemm_f8_blocks(d8, sd, wt8, swt)
        dw = ops.gemm_f8_blocks(dt8, sdt, xt8, sxt, out_dtype=torch.float32)
        return {'y': y, 'dx': dx, 'dw': dw}
    x, w, dy = x.float(), w.float(), dy.float()
    return {'y': (_blocks(x, 'e4m3')[0] @ _blocks(w, 'e4m3', 128)[0].T).bfloat16(),
            'dx': (_blocks(dy, s['grad'])[0] @ _blocks(w.T, 'e4m3', 128)[0].T).bfloat16(),
            'dw': _blocks(dy.T, s['grad'])[0] @ _blocks(x.T, 'e4m3')[0].T}


def _run_clip(s):
    if own:
        from merlot_amd import ops
        return {'norm': ops.clip_by_global_norm(s['list'], s['clip'], out=s['out_list']), 'grads': s['flat']}
    norm = torch.stack([t.double().square().sum() for t in s['grads']]).sum().sqrt().float()
    coef = s['clip'] / norm.clamp(min=s['clip'])
    [o.copy_(t.float() * coef) for o, t in zip(s['outs'], s['grads'])]
    return {'norm': norm, 'grads': s['flat']}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------

def work(case):
    op = case['op']
    if op == 'norm':
        n, e, res = case['rows'] * case['H'], 2 if case['dtype'] == 'bf16' else 4, case['residual']
        passes = (4 if res else 2) + (3 if case['backward'] else 0)      # x, residual -> h, y; dy, dh -> dx
        return {'bytes': passes * n * e + case['H'] * (8 if case['backward'] else 4), 'flops': (16 if case['backward'] else 5) * n}
    if op == 'chain':
        M, N, K = case['rows'], case['N'], case['H']
        return {'bytes': 6 * M * K + N * K + 2 * M * N, 'flops': 2 * M * N * K}
    if op == 'product':
        M, N, K = case['M'], case['N'], case['K']
        return {'bytes': (M + N) * (K + (K + 127) // 128) + (4 if case['out'] == 'f32' else 2) * M * N, 'flops': 2 * M * N * K}
    if op == 'linear':
        M, N, K = case['M'], case['N'], case['K']
        return {'bytes': 2 * (M * K + N * K + M * N) + 2 * (M * N + M * K) + 4 * N * K, 'flops': 6 * M * N * K}
    sizes = _sizes(case)
    n16 = sum(n for i, n in enumerate(sizes) if case['mixed'] and i % 4 == 1)
    n = sum(sizes)
    return {'bytes': 4 * (n - n16) + 2 * n16 + 4 * n, 'flops': 3 * n}


# ---- the operators' definitions in 64 bits -----------------------------------------------------------------------------------

def _power(e):
    """2^e in 64 bits, exactly"""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _quantized64(x, fmt, tile=1):
    """the values the blocks of x [R, C] (64 bits) stand for: nearest value of the format, ties to even, under the block's power of two"""
    mant, low, top = (3, -6, 448.0) if fmt == 'e4m3' else (2, -14, 57344.0)
    R, C = x.shape
    out = torch.zeros(_pad128(R) if tile > 1 else R, _pad128(C), dtype=torch.float64, device=x.device)
    out[:R, :C] = x
    v = out.view(-1, tile, _pad128(C) // 128, 128)
    amax = v.abs().amax((1, 3), keepdim=True)
    two = _power(torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, top)) / top)))
    two = torch.where(amax > two * top, two * 2, two)          # the logarithm's own rounding, next to a power of two
    two = torch.where(amax <= two / 2 * top, two / 2, two)
    u = v / two
    frac, e = torch.frexp(u.abs().clamp(min=2.0 ** low))
    step = _power(e - 1 - mant)
    return (torch.round(u / step) * step * two).view(out.shape)[:R]


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op in ('norm', 'chain'):
        x, g = s['x'].double(), s['gamma'].double()
        h = s['x'].double() if 'res' not in s else (x + s['res'].double()).to(s['x'].dtype).double()
        rms = (h.pow(2).sum(1, keepdim=True) / case['H'] + EPS).sqrt()
        n = h / rms
        if op == 'chain':
            w = s['w'].double() * _power(s['sw'].long() - 127).repeat_interleave(128, 1)
            return {'h': h, 'out': _quantized64(n * g, 'e4m3') @ w.t().contiguous()}
        out = {'y': n * g}
        if case['residual']:
            out['h'] = h
        if case['backward']:
            dy = s['dy'].double()
            dn = dy * g
            out['dx'] = (dn - n * (dn * n).sum(1, keepdim=True) / case['H']) / rms + s['dh'].double()
            out['dgamma'] = (dy * n).sum(0)
        return out
    if op == 'product':
        a, b = (s[k].double() * _power(s['s' + k].long() - 127).repeat_interleave(128, 1) for k in 'ab')
        c = a @ b.t().contiguous()
        return c if s['bias'] is None else c + s['bias'].double()
    if op == 'linear':
        x, w, dy = s['x'].double(), s['w'].double(), s['dy'].double()
        q = _quantized64
        return {'y': q(x, 'e4m3') @ q(w, 'e4m3', 128).t().contiguous(),
                'dx': q(dy, case['grad']) @ q(w.t(), 'e4m3', 128).t().contiguous(),
                'dw': q(dy.t(), case['grad']) @ q(x.t(), 'e4m3').t().contiguous()}
    total = sum(float(t.double().pow(2).sum()) for t in s['grads'])
    norm = math.sqrt(total)
    k = case['clip'] / max(norm, case['clip'])
    return {'norm': torch.tensor(norm, dtype=torch.float64, device='cuda'), 'grads': torch.cat([t.double() * k for t in s['grads']])}
