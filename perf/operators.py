"""The gated dense block and the 8-bit activation checkpoints, case by case: inputs, the plain torch form, the framework's calls.

  gated     H = act(X.Wg + bg) * (X.Wu + bu)                              the block's forward, alone (predict)
  train     the forward and its whole backward                           one training step's share of the block
  bwd       dX, dWg, dWu, dbg, dbu from dH and the kept G, U             the backward alone
  bwd8      the same with X, G, U kept in 8 bits                         the backward from checkpoints
  wgrad8    dW = X^T.dZ with X kept in 8 bits                            a dense layer's weight gradient from its checkpoint
  pack      values -> 8-bit checkpoint -> the values it stands for       writing and reading a checkpoint

The checkpoint's format: blocks of 32 consecutive values of a row share a power-of-two scale (one byte: exponent + 127), the values are
e4m3 codes of value / scale; the scale is the smallest power of two, 2^-126 at least, with max|value| <= 448 * scale; a block with a value
that is not finite stands for NaN throughout."""
import math

import numpy as np
import torch

own = False

BLOCK = 32


# ---- cases --------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a served model: latency, the weights' bytes are all there is to move
        dict(name='gated-1x1024x4096-bf16', op='gated', rows=1, fin=1024, units=4096, act='silu', dtype='bf16', bias=False),
        # a few nodes asked for at the width of this repository's models
        dict(name='gated-7x300x300-f32', op='gated', rows=7, fin=300, units=300, act='sigmoid', dtype='f32', bias=True),
        # predict over the smaller graph of the repository (9,475 nodes), 300 -> 600
        dict(name='gated-9475x300x600-f32', op='gated', rows=9475, fin=300, units=600, act='silu', dtype='f32', bias=True),
        # a wide block over a long batch, the largest product here
        dict(name='gated-8192x2048x8192-bf16', op='gated', rows=8192, fin=2048, units=8192, act='silu', dtype='bf16', bias=False),
        # the repository's 900 / 930-wide run over its 5,685 training nodes: odd widths, forward and backward
        dict(name='train-5685x900x930-f32', op='train', rows=5685, fin=900, units=930, act='gelu', dtype='f32', bias=True),
        # a whole step over the large graph of the repository (440,000 nodes, 300 wide)
        dict(name='train-440000x300x300-f32', op='train', rows=440000, fin=300, units=300, act='tanh', dtype='f32', bias=True),
        # the backward of a bf16 block over a long batch
        dict(name='bwd-8192x1024x4096-bf16', op='bwd', rows=8192, fin=1024, units=4096, act='silu', dtype='bf16', bias=False),
        # the large graph's backward with X, G, U kept in 8 bits
        dict(name='bwd8-440000x300x300-f32', op='bwd8', rows=440000, fin=300, units=300, act='sigmoid', dtype='f32', bias=True),
        # ... and a bf16 block's, one row more than whole tiles have
        dict(name='bwd8-4097x1024x1536-bf16', op='bwd8', rows=4097, fin=1024, units=1536, act='gelu', dtype='bf16', bias=True),
        # a plain dense layer's weight gradient from its 8-bit input: the output layer of the large graph's model
        dict(name='wgrad8-440000x300x256-f32', op='wgrad8', rows=440000, fin=300, units=256, act='none', dtype='f32', bias=False),
        # one activation of the smaller graph
        dict(name='pack-9475x300-f32', op='pack', rows=9475, fin=300, units=0, act='none', dtype='f32', bias=False),
        # one 600-wide activation of the large graph
        dict(name='pack-440000x600-f32', op='pack', rows=440000, fin=600, units=0, act='none', dtype='f32', bias=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = [work(c) for c in listed()]
    max_b, max_f = max(w['bytes'] for w in top), max(w['flops'] for w in top)
    while True:
        op = rng.choice(['gated', 'gated', 'train', 'bwd', 'bwd8', 'wgrad8', 'pack'])
        c = dict(op=op, rows=_log_int(rng, 1, 440000), fin=_log_int(rng, 33, 4096), units=0 if op == 'pack' else _log_int(rng, 33, 8192),
                 act='none' if op in ('wgrad8', 'pack') else rng.choice(['silu', 'gelu', 'sigmoid', 'tanh', 'relu', 'none']),
                 dtype=rng.choice(['f32', 'bf16']) if op != 'train' else 'f32', bias=rng.random() < 0.5)
        if op in ('wgrad8', 'pack'):
            c['bias'] = False
        w = work(c)
        if w['bytes'] <= max_b and w['flops'] <= max_f:
            return c


def work(case):
    M, K, N = case['rows'], case['fin'], case['units']
    s = 4 if case['dtype'] == 'f32' else 2
    q = 1 + 1 / BLOCK                                   # bytes of a value in a checkpoint
    op = case['op']
    vec = 8 * N if case['bias'] else 0                  # two fp32 bias vectors (or their gradients)
    if op == 'gated':
        return {'bytes': s * (M * K + 2 * K * N + M * N) + vec, 'flops': 4 * M * K * N}
    if op == 'train':                                   # X, dH, W in; H, dX, dW out
        return {'bytes': s * (2 * M * K + 2 * M * N + 4 * K * N) + 2 * vec, 'flops': 12 * M * K * N}
    if op == 'bwd':                                     # X, dH, G, U, W in; dX, dW out
        return {'bytes': s * (2 * M * K + 3 * M * N + 4 * K * N) + vec, 'flops': 8 * M * K * N}
    if op == 'bwd8':
        return {'bytes': q * (M * K + 2 * M * N) + s * (M * K + M * N + 4 * K * N) + vec, 'flops': 8 * M * K * N}
    if op == 'wgrad8':
        return {'bytes': q * M * K + s * (M * N + K * N), 'flops': 2 * M * K * N}
    return {'bytes': (2 * s + q) * M * K, 'flops': 8 * M * K}


# ---- inputs --------------------------------------------------------------------------------------------------------------------------
def _up(n, m):
    return (n + m - 1) // m * m


def _matrix(gen, n, F, dtype, scale, uniform=False):
    """Row-major with the framework's pitch for this type (roundup4 floats / roundup64 bf16), pad columns zero."""
    ld = _up(F, 4) if dtype == 'f32' else _up(F, 64)
    t = torch.zeros((n, ld), dtype=torch.float32 if dtype == 'f32' else torch.bfloat16, device='cuda')
    v = torch.rand((n, F), generator=gen, device='cuda') * 2 - 1 if uniform else torch.randn((n, F), generator=gen, device='cuda')
    t[:, :F] = v * scale
    return t


def _pow2(e):
    """2^e for integer tensors e in [-126, 127], from its bits."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _blocks(x):
    n, F = x.shape
    Fp = _up(F, BLOCK)
    if Fp != F:
        x = torch.nn.functional.pad(x, (0, Fp - F))
    return x.reshape(n, Fp // BLOCK, BLOCK)


def _quantise(x):
    """-> (values of the codes [n, blocks, 32], scale exponents [n, blocks], finite [n, blocks])"""
    b = _blocks(x.float())
    amax = b.abs().amax(dim=2)
    ok = torch.isfinite(amax)
    m, e = torch.frexp(torch.where(ok, amax, torch.zeros_like(amax)))
    s = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    y = torch.where(ok[:, :, None], b, torch.zeros_like(b)) * _pow2(-s)[:, :, None]
    _, ey = torch.frexp(y)
    step = (ey - 1).clamp(min=-6) - 3                    # e4m3: 3 bits behind the leading one, exponents from -6
    return torch.round(y * _pow2(-step)) * _pow2(step), s, ok


def _dequantise(q, s, ok, F):
    v = q * _pow2(s)[:, :, None]
    v = torch.where(ok[:, :, None], v, torch.full_like(v, float('nan')))
    return v.reshape(v.shape[0], -1)[:, :F]


def _codes(x):
    """The checkpoint as the framework stores it: codes [n, roundup32(F)] and scale bytes [n, roundup32(F) / 32]."""
    q, s, ok = _quantise(x)
    codes = q.to(torch.float8_e4m3fn).view(torch.uint8).reshape(x.shape[0], -1).contiguous()
    return codes, torch.where(ok, s + 127, torch.full_like(s, 255)).to(torch.uint8).contiguous()


def _read_codes(c, F):
    codes, scales = c
    s = scales.to(torch.int32)
    q = codes.view(torch.float8_e4m3fn).float().reshape(codes.shape[0], -1, BLOCK)
    return _dequantise(q, torch.where(s == 255, torch.zeros_like(s), s - 127), s != 255, F)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    M, K, N, dt, op = case['rows'], case['fin'], case['units'], case['dtype'], case['op']
    st = dict(case=case, x=_matrix(gen, M, K, dt, 0.5))
    if op not in ('wgrad8', 'pack'):
        for w in ('wg', 'wu'):
            st[w] = _matrix(gen, K, N, dt, math.sqrt(6.0 / (K + N)), uniform=True)
        for b in ('bg', 'bu'):
            st[b] = torch.randn(_up(N, 4), generator=gen, device='cuda') * 0.1 if case['bias'] else None
    if op in ('train', 'bwd', 'bwd8'):
        st['dh'] = _matrix(gen, M, N, dt, 1e-3)
    if op in ('bwd', 'bwd8'):
        st['g'], st['u'] = _matrix(gen, M, N, dt, 0.8), _matrix(gen, M, N, dt, 0.8)
    if op == 'wgrad8':
        st['dh'] = _matrix(gen, M, N, dt, 1e-3)
    if op in ('bwd8', 'wgrad8'):
        for k, F in (('x', K), ('g', N), ('u', N)):
            if k in st:
                st[k + '8'] = _codes(st.pop(k)[:, :F])
    if own:
        from geographconv_amd import ops
        mat = ops.DMat if dt == 'f32' else ops.HMat
        for k, n, F in (('x', M, K), ('wg', K, N), ('wu', K, N), ('dh', M, N), ('g', M, N), ('u', M, N)):
            if st.get(k) is not None:
                st[k] = mat(n, F, t=st[k])
            if k + '8' in st:
                st[k] = ops.MX8Mat(n, F, codes=st[k + '8'][0], scales=st[k + '8'][1], bf16=dt == 'bf16')
        st['act'] = {'silu': ops.ACT_SILU, 'gelu': ops.ACT_GELU, 'sigmoid': ops.ACT_SIGMOID, 'tanh': ops.ACT_TANH, 'relu': ops.ACT_RELU,
                     'none': ops.ACT_NONE}[case['act']]
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _out(m):
    return m.t[:, :m.F]


def _run_own(st):
    from geographconv_amd import ops
    c = st['case']
    op, N = c['op'], c['units']
    if op == 'gated':
        return _out(ops.gated_dense(st['x'], st['wg'], st['wu'], st['bg'], st['bu'], act=st['act']))
    if op == 'pack':
        return _out(ops.mx8_unpack(ops.mx8_pack(st['x'])))
    if op == 'wgrad8':
        return _out(ops.mx8_weight_grad(st['x'], st['dh']))
    h = None
    if op == 'train':
        h, kept = ops.gated_dense(st['x'], st['wg'], st['wu'], st['bg'], st['bu'], act=st['act'], keep='full')
    else:
        kept = ops.GatedTape(st['g'], st['u'])
    dx, dwg, dwu, dbg, dbu = ops.gated_dense_bwd(st['dh'], st['x'], st['wg'], st['wu'], kept, act=st['act'], bias=c['bias'])
    res = dict(dx=_out(dx), dwg=_out(dwg), dwu=_out(dwu))
    if c['bias']:
        res.update(dbg=dbg[:N], dbu=dbu[:N])
    if h is not None:
        res['h'] = _out(h)
    return res


def _act(a, x):
    if a == 'silu':
        return x / (1 + torch.exp(-x))
    if a == 'gelu':
        return x * 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
    if a == 'sigmoid':
        return 1 / (1 + torch.exp(-x))
    if a == 'tanh':
        return torch.tanh(x)
    if a == 'relu':
        return torch.clamp(x, min=0)
    return x


def _act_grad(a, x):
    if a == 'silu':
        s = 1 / (1 + torch.exp(-x))
        return s * (1 + x * (1 - s))
    if a == 'gelu':
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    if a == 'sigmoid':
        s = 1 / (1 + torch.exp(-x))
        return s * (1 - s)
    if a == 'tanh':
        t = torch.tanh(x)
        return 1 - t * t
    if a == 'relu':
        return (x > 0).to(x.dtype)
    return torch.ones_like(x)


def _run_plain(st):
    c = st['case']
    op, K, N, a = c['op'], c['fin'], c['units'], c['act']
    odt = torch.float32 if c['dtype'] == 'f32' else torch.bfloat16
    if op == 'pack':
        q, s, ok = _quantise(st['x'][:, :K])
        return _dequantise(q, s, ok, K).to(odt)
    x = _read_codes(st['x8'], K) if 'x8' in st else st['x'][:, :K].float()
    if op == 'wgrad8':
        return (x.t() @ st['dh'][:, :N].float()).to(odt)
    wg, wu = st['wg'][:, :N].float(), st['wu'][:, :N].float()
    res = {}
    if op in ('gated', 'train'):
        g, u = x @ wg, x @ wu
        if c['bias']:
            g, u = g + st['bg'][:N], u + st['bu'][:N]
        h = (_act(a, g) * u).to(odt)
        if op == 'gated':
            return h
        res['h'] = h
    elif op == 'bwd':
        g, u = st['g'][:, :N].float(), st['u'][:, :N].float()
    else:
        g, u = _read_codes(st['g8'], N), _read_codes(st['u8'], N)
    dh = st['dh'][:, :N].float()
    dg, du = dh * u * _act_grad(a, g), dh * _act(a, g)
    res.update(dx=(dg @ wg.t() + du @ wu.t()).to(odt), dwg=(x.t() @ dg).to(odt), dwu=(x.t() @ du).to(odt))
    if c['bias']:
        res.update(dbg=dg.sum(0), dbu=du.sum(0))
    return res


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------------
def _e4m3_grid():
    """Every value of a finite, non-negative e4m3 code, in code order: 0, subnormals of 2^-9, then (8 + m) / 8 * 2^(e - 7); 448 is the last."""
    return np.array([(c % 8) / 8 * 2.0 ** -6 if c < 8 else (1 + (c % 8) / 8) * 2.0 ** (c // 8 - 7) for c in range(127)])


def _checkpoint64(x):
    """The values the checkpoint of x stands for: nearest grid point of value / scale, a tie to the even code."""
    grid = torch.from_numpy(_e4m3_grid()).cuda()
    mid = (grid[1:] + grid[:-1]) / 2
    n, F = x.shape
    out = torch.empty((n, F), dtype=torch.float64, device='cuda')
    step = max(1, (1 << 25) // max(F, 1))
    for r in range(0, n, step):
        v = x[r:r + step].double()
        w = torch.zeros((v.shape[0], _up(F, BLOCK)), dtype=torch.float64, device='cuda')
        w[:, :F] = v
        w = w.view(v.shape[0], -1, BLOCK)
        top = w.abs().amax(-1, keepdim=True)
        bad = ~torch.isfinite(top)
        scale = torch.full_like(top, 2.0 ** -126)
        for _ in range(2):                               # the power of two at or above top / 448, from the bits of the quotient
            e = ((top / 448).view(torch.int64) >> 52) - 1023
            e = torch.where((e.double() >= -126) & ~bad, e, torch.full_like(e, -126))
            p = ((e + 1023) << 52).view(torch.float64)
            scale = torch.where(p * 448 >= top, p, p * 2)
        r_ = w.abs() / scale
        r_ = torch.where(bad, torch.zeros_like(r_), r_)
        lo = torch.searchsorted(mid, r_.contiguous())    # first midpoint >= r: code lo, or lo + 1 on a tie with odd lo
        tie = (lo < len(mid)) & (mid[lo.clamp(max=len(mid) - 1)] == r_) & (lo % 2 == 1)
        val = grid[lo + tie.long()] * scale * torch.sign(w)
        val = torch.where(bad, torch.full_like(val, float('nan')), val)
        out[r:r + step] = val.view(v.shape[0], -1)[:, :F]
    return out


def _sigma64(x):
    return torch.special.expit(x)


def _gate64(a, g):
    """(act(g), act'(g)) in 64 bits"""
    if a == 'silu':
        s = _sigma64(g)
        return g * s, s + g * s * _sigma64(-g)
    if a == 'gelu':
        cdf = torch.special.ndtr(g)
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if a == 'sigmoid':
        s = _sigma64(g)
        return s, s * _sigma64(-g)
    if a == 'tanh':
        return torch.tanh(g), 1 / torch.cosh(g) ** 2
    if a == 'relu':
        return g * (g > 0), (g > 0).double()
    return g, torch.ones_like(g)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    op, K, N = case['op'], case['fin'], case['units']
    if op == 'pack':
        return _checkpoint64(st['x'][:, :K])

    def kept(k, F):
        if k in st:
            return st[k][:, :F].double()
        codes, scales = st[k + '8']
        mag = torch.from_numpy(np.concatenate([_e4m3_grid(), [np.nan]])).cuda()
        full = torch.cat([mag, -mag])[codes.long()]
        e = scales.long()
        sc = torch.where(e == 255, torch.full_like(e, 2047 << 52) + 1, (e - 127 + 1023) << 52).view(torch.float64)
        return (full.view(codes.shape[0], -1, BLOCK) * sc[:, :, None]).view(codes.shape[0], -1)[:, :F].contiguous()

    x = kept('x', K)
    if op == 'wgrad8':
        return torch.mm(x.t(), st['dh'][:, :N].double())
    wg, wu = st['wg'][:, :N].double(), st['wu'][:, :N].double()
    if op in ('gated', 'train'):
        g, u = torch.mm(x, wg), torch.mm(x, wu)
        if case['bias']:
            g += st['bg'][:N].double()
            u += st['bu'][:N].double()
    else:
        g, u = kept('g', N), kept('u', N)
    value, slope = _gate64(case['act'], g)
    if op == 'gated':
        return value * u
    dh = st['dh'][:, :N].double()
    dg, du = slope * u * dh, value * dh
    res = {}
    if op == 'train':
        res['h'] = value * u
    res['dx'] = torch.mm(dg, wg.t()) + torch.mm(du, wu.t())
    res['dwg'], res['dwu'] = torch.mm(x.t(), dg), torch.mm(x.t(), du)
    if case['bias']:
        res['dbg'], res['dbu'] = dg.sum(0), du.sum(0)
    return res
