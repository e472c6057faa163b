"""The gated dense block and the 8-bit checkpoints where the sizes, types and values of test_gated_gpu.py do not reach (run on the MI355X:
pytest -m gpu).  Bounds: as derived there (ENV * sum|a.b| for a product, half a step for a stored result); what is added is stated at each test."""
import numpy as np
import pytest

from . import gated_reference as R, gated_shapes as S
from .test_gated_gpu import BF, ENV, EPS, _check, _f64, _forward_bounds, _mat, _problem, _rand

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    from geographconv_amd import ops
    ops.require_gpu()
    return torch.device("cuda:0")


@pytest.mark.parametrize('M,K,N,eight', [(1, 33, 40, False), (130, 40, 300, False), (700, 1100, 200, True), (5000, 96, 161, True), (4097, 600, 530, False)])
def test_bf16_gradients_are_rounded_once(dev, M, K, N, eight):
    """dG and dU of a bf16 block are fp32 values; multiplied as two bf16 terms they are off by 2^-16, so a gradient is off by its own rounding
    (half a step, 2^-8 of it) and 2^-16 of the products' magnitudes.  precision='bf16': one term, 2^-8 of the magnitudes."""
    from geographconv_amd import ops
    d, r = _problem(dev, M, K, N, 'bf16', False, M + N)
    G, U = _mat(_rand((M, N), 21), dev, 'bf16'), _mat(_rand((M, N), 22), dev, 'bf16')
    dH = _mat(_rand((M, N), 23, 1e-3), dev, 'bf16')
    X = d['X']
    if eight:
        X, G, U = ops.mx8_pack(X), ops.mx8_pack(G), ops.mx8_pack(U)
    read = lambda m: _f64(ops.mx8_unpack(m)) if eight else _f64(m)
    x, g, u, h = read(X), read(G), read(U), _f64(dH)
    dG, dU = R.gate_grads(h, g, u, 'silu')
    eg, eu = EPS * (1 + np.abs(g)) * np.abs(h * u) + 1e-37, EPS * (1 + np.abs(g)) * np.abs(h) + 1e-37
    wg, wu, ax = np.abs(r['Wg']), np.abs(r['Wu']), np.abs(x).T
    want = dict(dX=(dG @ r['Wg'].T + dU @ r['Wu'].T, np.abs(dG) @ wg.T + np.abs(dU) @ wu.T, eg @ wg.T + eu @ wu.T),
                dWg=(x.T @ dG, ax @ np.abs(dG), ax @ eg), dWu=(x.T @ dU, ax @ np.abs(dU), ax @ eu))
    for precision, terms in ((None, 2.0 ** -16), ('f32', 2.0 ** -16), ('bf16', BF)):
        res = ops.gated_dense_bwd(dH, X, d['Wg'], d['Wu'], ops.GatedTape(G, U), act=ops.ACT_SILU, precision=precision)
        for m, (name, (w, mag, e)) in zip(res, want.items()):
            _check(_f64(m), (w, (1 + BF) * ((ENV + terms) * mag + 2 * e) + BF * np.abs(w) + 1e-30), '%s %s' % (name, precision))


TOP = 240 * 2.0 ** 120          # the largest number that a checkpoint of finite values stands for: the next code at this scale is 2^128


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_the_largest_values_stay_finite(dev, dtype):
    """Finite values up to the type's largest read back finite, off by 2^-4 of themselves at most, their block's other values too."""
    from geographconv_amd import ops
    big = torch.finfo(torch.float32 if dtype == 'f32' else torch.bfloat16).max
    x = np.zeros((4, 64))
    x[0, :6] = [big, -big, 3.3e38, 1.9375 * 2.0 ** 127, 2.0 ** 127, 2.0 ** 125]
    x[1, :3] = [1.875 * 2.0 ** 127, -1.75 * 2.0 ** 127, 1.5 * 2.0 ** 118]
    x[2, 33:35] = [-1.9375 * 2.0 ** 127, 3e37]
    x[3] = big
    m = _mat(x.astype(np.float32), dev, dtype)
    q = ops.mx8_pack(m)
    x = _f64(m)
    got = _f64(ops.mx8_unpack(q))
    s = 2.0 ** (np.repeat(q.scales.cpu().numpy().astype(np.float64), 32, axis=1) - 127)
    _check(got, (x, np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s)), 'checkpoint')
    want = np.clip(R.mx8(x)[2], -TOP, TOP)
    assert np.array_equal(got, want)


@pytest.mark.parametrize('M,K', [(1, 1), (5, 40), (300, 40), (40, 4096)])
def test_the_largest_pre_activations_stay_finite_in_their_checkpoints(dev, M, K):
    """... in the checkpoints that the block's forward writes: a few rows, tiles, a split reduction."""
    from geographconv_amd import ops
    big = float(torch.finfo(torch.bfloat16).max)
    X, Wg, Wu = np.zeros((M, K), np.float32), np.zeros((K, 40), np.float32), np.zeros((K, 40), np.float32)
    X[:, 0] = 1
    Wg[0, ::3], Wg[0, 1::3], Wu[0] = big, -2.0 ** 126, 0.5
    _, kept = ops.gated_dense(*(_mat(a, dev, 'bf16') for a in (X, Wg, Wu)), act=ops.ACT_NONE, keep='mx8')
    got = _f64(ops.mx8_unpack(kept.G))
    assert np.array_equal(got, np.tile(np.clip(R.mx8(Wg[:1].astype(np.float64))[2], -TOP, TOP), (M, 1)))


def _poisoned(n, F, ld, dtype, dev):
    from geographconv_amd import ops
    t = torch.full((n, ld), float('nan'), dtype=torch.float32 if dtype == 'f32' else torch.bfloat16, device=dev)
    return (ops.DMat if dtype == 'f32' else ops.HMat)(n, F, t=t)


def _check_pads(m, what):
    """The pad columns of a result: zero up to roundup4 (fp32) / roundup64 or the pitch (bf16), left alone behind."""
    from geographconv_amd import ops
    end = ops.pad4(m.F) if isinstance(m, ops.DMat) else min(m.ld, (m.F + 63) // 64 * 64)
    assert torch.isfinite(m.t[:, :end].float()).all(), what
    assert (m.t[:, m.F:end] == 0).all() and torch.isnan(m.t[:, end:].float()).all(), what


def _forward_into(X, Wg, Wu, act, H, keep, G, U, precision):
    """The C entry with given matrices for the kept G, U."""
    from geographconv_amd import _ffi, ops
    ops._on_device(H.t.get_device(), ops._call_with_ws, _ffi.lib().geogcn_gated_fwd, 'gated_fwd', X.n, X.F, Wg.F, ops._mat_type(X), X.t.data_ptr(), X.ld,
                   Wg.t.data_ptr(), Wg.ld, Wu.t.data_ptr(), Wu.ld, None, None, act, H.t.data_ptr(), H.ld, ops._KEEP[keep], *ops._mat_args(G),
                   *ops._mat_args(U), ops.GEMM_PRECISIONS[precision])


@pytest.mark.parametrize('M,K', [(5, 70), (300, 70), (40, 4096)])
def test_kept_matrices_of_other_pitches_have_zero_pads(dev, M, K):
    """bf16 G and U of wider pitches than H's: their own pads are zero too (a few rows, tiles, a split reduction)."""
    from geographconv_amd import ops
    N = 90
    d, r = _problem(dev, M, K, N, 'bf16', False, M)
    for lds in ((92, 128, 96), (92, 92, 200), (128, 128, 128)):
        H, G, U = (_poisoned(M, N, ld, 'bf16', dev) for ld in lds)
        _forward_into(d['X'], d['Wg'], d['Wu'], ops.ACT_SILU, H, 'full', G, U, 'bf16x3')
        for m, ref, what in zip((H, G, U), _forward_bounds(r, 'silu', 'bf16'), 'HGU'):
            _check(_f64(m), ref, what)
            _check_pads(m, (what, lds))


@pytest.mark.parametrize('M', [30, 3000])
@pytest.mark.parametrize('precision', ['bf16x3', 'bf16'])
def test_weight_gradients_of_other_pitches_have_zero_pads(dev, M, precision):
    from geographconv_amd import ops
    K, N = 70, 90
    d, r = _problem(dev, M, K, N, 'bf16', False, M)
    kept = ops.GatedTape(_mat(_rand((M, N), 21), dev, 'bf16'), _mat(_rand((M, N), 22), dev, 'bf16'))
    dH = _mat(_rand((M, N), 23), dev, 'bf16')
    want = ops.gated_dense_bwd(dH, d['X'], d['Wg'], d['Wu'], kept, act=ops.ACT_SILU, precision=precision)
    for lds in ((128, 92), (92, 128), (96, 200)):
        dX, dWg, dWu = _poisoned(M, K, 72, 'bf16', dev), *(_poisoned(K, N, ld, 'bf16', dev) for ld in lds)
        ops.gated_dense_bwd(dH, d['X'], d['Wg'], d['Wu'], kept, act=ops.ACT_SILU, dX=dX, dWg=dWg, dWu=dWu, precision=precision)
        for m, w, what in zip((dX, dWg, dWu), want, ('dX', 'dWg', 'dWu')):
            assert torch.equal(m.t[:, :m.F], w.t[:, :m.F])
            _check_pads(m, (what, lds))


# ---- every tile shape, every result ------------------------------------------------------------------------------------------------------------
# Inputs of the blocks at precision='bf16' are numbers that bf16 holds, so rounding the operands changes nothing and the bounds above stand; dG and
# dU are not, and are off by half a step (BF).  References: torch's products of 64-bit matrices, on the GPU.
def _mat_on(gen, n, F, dtype, scale, precision, dev, ld=None):
    from geographconv_amd import ops
    v = torch.randn((n, F), generator=gen, device=dev) * scale
    if precision == 'bf16':
        v = v.bfloat16().float()
    ld = ld or (ops.pad4(F) if dtype == 'f32' else ops.bf16_ld(F))
    t = torch.zeros((n, ld), dtype=torch.float32 if dtype == 'f32' else torch.bfloat16, device=dev)
    t[:, :F] = v
    return (ops.DMat if dtype == 'f32' else ops.HMat)(n, F, t=t)


def _wide(m):
    """the values of a matrix or a checkpoint in 64 bits, on the GPU"""
    from geographconv_amd import ops
    m = ops.mx8_unpack(m) if isinstance(m, ops.MX8Mat) else m
    return m.t[:, :m.F].double().contiguous()


def _close(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    bad = (got - want).abs() > bound
    assert not bad.any(), "%s: %d of %d entries out of bounds, worst %.3g x" % (what, bad.sum(), bad.numel(), ((got - want).abs() / bound).max())


def _silu(g):
    s = torch.sigmoid(g)
    return g * s, s * (1 + g * (1 - s))


def _seeded(dev, *sizes):
    return torch.Generator(device=dev).manual_seed(sum(s * p for s, p in zip(sizes, (1, 3, 7))))


@pytest.mark.parametrize('M,K,N,dtype,precision', S.FORWARD)
def test_forward_on_every_tile_shape(dev, M, K, N, dtype, precision):
    from geographconv_amd import ops
    gen = _seeded(dev, M, K, N)
    X = _mat_on(gen, M, K, dtype, 1.0, precision, dev)
    Wg, Wu = (_mat_on(gen, K, N, dtype, K ** -0.5, precision, dev) for _ in range(2))
    b = [torch.randn(N, generator=gen, device=dev) for _ in range(2)]
    x, wg, wu = _wide(X), _wide(Wg), _wide(Wu)
    G, U = x @ wg + b[0].double(), x @ wu + b[1].double()
    eg, eu = (ENV * (x.abs() @ w.abs() + v.double().abs()) for w, v in ((wg, b[0]), (wu, b[1])))
    v = _silu(G)[0]
    half = BF if dtype == 'bf16' else 2.0 ** -23
    h = 1.2 * U.abs() * eg + v.abs() * eu + EPS * v.abs() * U.abs() + EPS * U.abs() + half * (v * U).abs() + 1e-30
    out = _poisoned(M, N, ops.pad4(N) + 4 if dtype == 'f32' else ops.bf16_ld(N), dtype, dev)
    H, kept = ops.gated_dense(X, Wg, Wu, *b, act=ops.ACT_SILU, keep='full', precision=precision, out=out)
    _close(H.t[:, :N], v * U, h, 'H')
    _check_pads(H, 'H')
    for m, w, e, what in ((kept.G, G, eg, 'G'), (kept.U, U, eu, 'U')):
        _close(m.t[:, :N], w, e + half * w.abs() + 1e-30, what)
        assert (m.t[:, N:ops.pad4(N) if dtype == 'f32' else m.ld] == 0).all(), what
    H8, k8 = ops.gated_dense(X, Wg, Wu, *b, act=ops.ACT_SILU, keep='mx8', precision=precision)
    _close(H8.t[:, :N], v * U, h, 'H beside checkpoints')
    _close(ops.gated_dense(X, Wg, Wu, *b, act=ops.ACT_SILU, precision=precision).t[:, :N], v * U, h, 'H alone')
    for q, w, e, what in ((k8.G, G, eg, 'G'), (k8.U, U, eu, 'U')):
        s = torch.exp2(q.scales.double() - 127).repeat_interleave(32, dim=1)[:, :N]
        got = _wide(q)
        _close(got, w, torch.maximum(2.0 ** -4 * (w.abs() + e), 2.0 ** -10 * s) * (1 + 1e-6) + e + (BF * w.abs() if dtype == 'bf16' else 0), what + ' in 8 bits')
        assert (q.codes[:, N:] & 0x7f == 0).all()


def _backward_case(dev, M, K, N, dtype, precision, eight):
    from geographconv_amd import ops
    gen = _seeded(dev, M, K, N)
    X = _mat_on(gen, M, K, dtype, 1.0, precision, dev)
    Wg, Wu = (_mat_on(gen, K, N, dtype, K ** -0.5, precision, dev) for _ in range(2))
    G, U = (_mat_on(gen, M, N, dtype, 1.0, None, dev) for _ in range(2))
    dH = _mat_on(gen, M, N, dtype, 1e-3, None, dev)
    if eight:
        X, G, U = ops.mx8_pack(X), ops.mx8_pack(G), ops.mx8_pack(U)
    x, wg, wu, g, u, h = (_wide(m) for m in (X, Wg, Wu, G, U, dH))
    v, d = _silu(g)
    dG, dU = h * u * d, h * v
    eg, eu = EPS * (1 + g.abs()) * (h * u).abs() + 1e-37, EPS * (1 + g.abs()) * h.abs() + 1e-37
    rnd = ENV + (BF if precision == 'bf16' else 2.0 ** -16 if dtype == 'bf16' else 0)
    half = BF if dtype == 'bf16' else 2.0 ** -23
    xt, ax = x.t().contiguous(), x.t().abs().contiguous()
    want = [(dG @ wg.t().contiguous() + dU @ wu.t().contiguous(),
             (rnd * dG.abs() + 2 * eg) @ wg.t().abs().contiguous() + (rnd * dU.abs() + 2 * eu) @ wu.t().abs().contiguous()),
            (xt @ dG, ax @ (rnd * dG.abs() + 2 * eg)), (xt @ dU, ax @ (rnd * dU.abs() + 2 * eu))]
    want = [(w, (1 + half) * e + half * w.abs() + 1e-30) for w, e in want]
    want += [(t.sum(0), 128 * 2.0 ** -24 * t.abs().sum(0) + e.sum(0) + 1e-30) for t, e in ((dG, eg), (dU, eu))]
    ld = lambda F: ops.pad4(F) + 4 if dtype == 'f32' else ops.bf16_ld(F) + 8
    outs = [_poisoned(n, F, ld(F), dtype, dev) for n, F in ((M, K), (K, N), (K, N))]
    ops.gated_dense_bwd(dH, X, Wg, Wu, ops.GatedTape(G, U), act=ops.ACT_SILU, dX=outs[0], dWg=outs[1], dWu=outs[2], precision=precision)
    db = ops.gated_dense_bwd(dH, X, Wg, Wu, ops.GatedTape(G, U), act=ops.ACT_SILU, bias=True, need_input_grad=False, precision=precision)[3:]
    for m, (w, e), what in zip(outs, want, ('dX', 'dWg', 'dWu')):
        _close(m.t[:, :m.F], w, e, what)
        _check_pads(m, what)
    for t, (w, e), what in zip(db, want[3:], ('dbg', 'dbu')):
        _close(t[:N], w, e, what)


@pytest.mark.parametrize('M,K,N,dtype,precision,eight', S.BACKWARD)
def test_backward_on_every_tile_shape(dev, M, K, N, dtype, precision, eight):
    _backward_case(dev, M, K, N, dtype, precision, eight)


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('M,K,N,precision', [(16390, 301, 203, 'bf16x3'), (20000, 193, 65, 'bf16x3'), (70, 45, 33, 'f32'), (16390, 301, 203, 'f32'), (1, 5, 3, 'f32')])
def test_backward_on_the_librarys_kernels(dev, M, K, N, precision, eight):
    """... and on the library's whole-rows and A^T.B kernels, and its exact fp32 ones."""
    _backward_case(dev, M, K, N, 'f32', precision, eight)


@pytest.mark.parametrize('M,K,N,dtype,precision', S.WEIGHT + [(16500, 301, 255, 'f32', 'bf16x3'), (100, 901, 637, 'f32', 'bf16x3'), (300, 45, 33, 'f32', 'f32')])
def test_weight_gradient_on_every_tile_shape(dev, M, K, N, dtype, precision):
    from geographconv_amd import ops
    gen = _seeded(dev, M, K, N)
    X = ops.mx8_pack(_mat_on(gen, M, K, dtype, 1.0, None, dev))
    dZ = _mat_on(gen, M, N, dtype, 1e-2, precision, dev)
    x, z = _wide(X).t().contiguous(), _wide(dZ)
    out = _poisoned(K, N, ops.pad4(N) + 4 if dtype == 'f32' else ops.bf16_ld(N) + 8, dtype, dev)
    ops.mx8_weight_grad(X, dZ, out=out, precision=precision)
    want = x @ z
    _close(out.t[:, :N], want, ENV * (x.abs() @ z.abs()) + (BF if dtype == 'bf16' else 2.0 ** -23) * want.abs() + 1e-30, 'dW')
    _check_pads(out, 'dW')


# ---- calls that the tests of the sizes above do not make -----------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype,ld', [('f32', 160), ('bf16', 132), ('bf16', 136)])
@pytest.mark.parametrize('M', [1, 3, 9, 16])
def test_a_few_rows_with_junk_in_the_pads(dev, M, dtype, ld):
    """Pitches that allow wide loads and that do not, NaN behind roundup4(F) in every operand, a result among rows that stay as they were."""
    from geographconv_amd import ops
    K, N = 70, 90
    d, r = _problem(dev, M, K, N, dtype, True, 12, ld=ld, junk=True)
    kind = ops.DMat if dtype == 'f32' else ops.HMat
    big = torch.full((M + 4, ld), 7.0, dtype=torch.float32 if dtype == 'f32' else torch.bfloat16, device=dev)
    H, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=ops.ACT_GELU, keep='full', out=kind(M + 4, N, t=big).rows(2, M + 2))
    for m, ref in zip((H, kept.G, kept.U), _forward_bounds(r, 'gelu', dtype)):
        _check(_f64(m), ref, 'H, G, U')
    assert (big[:2] == 7).all() and (big[M + 2:] == 7).all()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('M,K,N', [(9, 70, 100), (300, 70, 100), (16400, 200, 100)])
def test_a_gradient_row_that_is_not_finite_stays_alone(dev, M, K, N, dtype):
    """An infinity or a NaN in a row of dH reaches that row of dX and no other."""
    from geographconv_amd import ops
    d, _ = _problem(dev, M, K, N, dtype, False, 6)
    kept = ops.GatedTape(_mat(_rand((M, N), 21), dev, dtype), _mat(_rand((M, N), 22), dev, dtype))
    dH = _mat(_rand((M, N), 23), dev, dtype)
    want = ops.gated_dense_bwd(dH, d['X'], d['Wg'], d['Wu'], kept)[0]
    dH.t[3, 5], dH.t[8, 99] = float('inf'), float('nan')
    got = ops.gated_dense_bwd(dH, d['X'], d['Wg'], d['Wu'], kept)[0]
    ok = torch.ones(M, dtype=torch.bool, device=dev)
    ok[[3, 8]] = False
    assert torch.equal(want.t[ok], got.t[ok])
    assert not torch.isfinite(got.t[~ok][:, :K].float()).any()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_matrices_of_more_than_2_31_values(dev, dtype):
    """8,500,000 x 256 -> 256: every offset passes 32 bits.  The last rows against 64 bits; the weight gradients against 64-bit sums in pieces."""
    from geographconv_amd import ops
    M, F = 8_500_000, 256
    kind, tdt = (ops.DMat, torch.float32) if dtype == 'f32' else (ops.HMat, torch.bfloat16)
    gen = torch.Generator(device=dev).manual_seed(1)

    def big(scale):
        t = torch.empty((M, F), dtype=tdt, device=dev)
        for i in range(0, M, 500_000):
            t[i:i + 500_000] = torch.randn((min(500_000, M - i), F), generator=gen, device=dev) * scale
        return kind(M, F, t=t)
    X, dH = big(1.0), big(1e-3)
    Wg, Wu = (kind(F, F, t=(torch.randn((F, F), generator=gen, device=dev) / 16).to(tdt)) for _ in range(2))
    H, kept = ops.gated_dense(X, Wg, Wu, act=ops.ACT_NONE, keep='full')
    x8 = ops.mx8_pack(X)
    dX, dWg, dWu, dbg, dbu = ops.gated_dense_bwd(dH, X, Wg, Wu, kept, act=ops.ACT_NONE, bias=True)
    d8 = ops.mx8_weight_grad(x8, dH)
    n = 300
    half = BF if dtype == 'bf16' else 2.0 ** -23
    rnd = ENV + (2.0 ** -16 if dtype == 'bf16' else 0)
    wide = lambda m, a, b: m.t[a:b].double()
    wg, wu = wide(Wg, 0, F), wide(Wu, 0, F)
    a = M - n
    x, h, g, u = (wide(m, a, M) for m in (X, dH, kept.G, kept.U))
    mg, mu = x.abs() @ wg.abs(), x.abs() @ wu.abs()
    for m, w, mag in ((kept.G, x @ wg, mg), (kept.U, x @ wu, mu)):
        _close(m.t[a:], w, ENV * mag + half * w.abs() + 1e-30, 'G, U')
    G, U = x @ wg, x @ wu
    _close(H.t[a:], G * U, 1.01 * (U.abs() * ENV * mg + G.abs() * ENV * mu) + (half + EPS) * (G * U).abs() + 1e-30, 'H')
    want = (h * u) @ wg.t().contiguous() + (h * g) @ wu.t().contiguous()
    mag = (h * u).abs() @ wg.t().abs().contiguous() + (h * g).abs() @ wu.t().abs().contiguous()
    _close(dX.t[a:], want, (rnd + EPS) * mag + half * want.abs() + 1e-30, 'dX')
    _close(ops.mx8_unpack(x8).t[a:], x, 2.0 ** -4 * x.abs() + 2.0 ** -10 * 2.0 ** -6, 'checkpoint')
    sums = [torch.zeros((F, F), dtype=torch.float64, device=dev) for _ in range(6)]
    cols = [torch.zeros(F, dtype=torch.float64, device=dev) for _ in range(4)]
    for i in range(0, M, 500_000):
        j = min(M, i + 500_000)
        x, h, g, u = (wide(m, i, j) for m in (X, dH, kept.G, kept.U))
        q = ops.mx8_unpack(ops.MX8Mat(j - i, F, x8.codes[i:j], x8.scales[i:j], dtype == 'bf16')).t.double()
        for k, (l, r) in enumerate(((x, h * u), (x, h * g), (q, h))):
            sums[2 * k] += l.t().contiguous() @ r
            sums[2 * k + 1] += l.t().abs().contiguous() @ r.abs()
        for k, r in enumerate((h * u, h * g)):
            cols[2 * k] += r.sum(0)
            cols[2 * k + 1] += r.abs().sum(0)
    for k, (m, e) in enumerate(((dWg, rnd), (dWu, rnd), (d8, ENV))):
        _close(m.t, sums[2 * k], (e + EPS) * sums[2 * k + 1] + half * sums[2 * k].abs(), ('dWg', 'dWu', 'dW from codes')[k])
    # (partial sums of at most 2,048 rows, then of at most 65,535 / 16 of those: far fewer than 2^12 additions in a row)
    for k, t in enumerate((dbg, dbu)):
        _close(t[:F], cols[2 * k], 2.0 ** 12 * 2.0 ** -24 * cols[2 * k + 1], 'bias')


@pytest.mark.parametrize('M,K,N,precision', [(5, 70, 91, 'bf16x3'), (300, 70, 91, 'bf16x3'), (16385, 301, 257, 'bf16x3'), (33000, 70, 645, 'bf16x3'), (300, 70, 91, 'f32'),
                                             (17000, 45, 33, 'f32'), (300, 70, 91, 'bf16'), (40, 2500, 91, 'bf16x3')])
def test_fp32_results_of_every_forward_route_have_zero_pads(dev, M, K, N, precision):
    """A few rows, tiles, split reductions, the library's whole-rows and exact kernels: H, G and U into matrices full of NaN."""
    from geographconv_amd import ops
    gen = _seeded(dev, M, K, N)
    X = _mat_on(gen, M, K, 'f32', 1.0, precision, dev)
    Wg, Wu = (_mat_on(gen, K, N, 'f32', K ** -0.5, precision, dev) for _ in range(2))
    x, wg, wu = _wide(X), _wide(Wg), _wide(Wu)
    G, U = x @ wg, x @ wu
    eg, eu = ENV * (x.abs() @ wg.abs()), ENV * (x.abs() @ wu.abs())
    v = _silu(G)[0]
    out = [_poisoned(M, N, ops.pad4(N) + e, 'f32', dev) for e in (4, 8, 4)]
    _forward_into(X, Wg, Wu, ops.ACT_SILU, out[0], 'full', out[1], out[2], precision)
    h = 1.2 * U.abs() * eg + v.abs() * eu + EPS * v.abs() * U.abs() + EPS * U.abs() + 1e-30
    for m, w, e, what in zip(out, (v * U, G, U), (h, eg, eu), 'HGU'):
        _close(m.t[:, :N], w, e + 2.0 ** -23 * w.abs() + 1e-30, what)
        _check_pads(m, what)
    H = _poisoned(M, N, ops.pad4(N), 'f32', dev)
    ops.gated_dense(X, Wg, Wu, act=ops.ACT_SILU, out=H, precision=precision)
    _close(H.t[:, :N], v * U, h + 2.0 ** -23 * (v * U).abs(), 'H alone')
    assert (H.t[:, N:] == 0).all()
