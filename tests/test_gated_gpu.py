"""The gated dense block and the 8-bit activation checkpoints through the C ABI against 64-bit NumPy (run on the MI355X: pytest -m gpu).

Tolerances.  A product of fp32 matrices (exact kernels or three bf16 terms a value) is held to the library's envelope ENV * sum|a.b|, a product of
bf16 matrices (exact products, fp32 accumulation) too; a result stored as bf16 adds half a step, 2^-8 of itself.  Through the gate:
|act'| <= 1.2 for every activation here, so |dH| <= 1.2 |u| dg + |act(g)| du + 2^-20 |act(g) u| (a few ulp of the functions) + 2^-20 |u| (the
absolute error of a saturated one).  Gate gradients: 2^-20 (1 + |g|) |dh u| and 2^-20 (1 + |g|) |dh| absolute (the derivative's cancellation),
summed with the other factor's magnitude in the products; in a bf16 block each is also rounded once (2^-8)."""
import numpy as np
import pytest

from . import gated_reference as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ENV = 2e-6
BF = 2.0 ** -8
EPS = 2.0 ** -20


@pytest.fixture(scope="module")
def dev():
    from geographconv_amd import ops
    ops.require_gpu()
    return torch.device("cuda:0")


def _rand(shape, seed, scale=1.0):
    return (np.random.RandomState(seed).randn(*shape) * scale).astype(np.float32)


def _mat(a, dev, dtype, ld=None, junk=False):
    """A DMat / HMat of `a`; junk: the pad columns behind roundup4 hold NaN (the convention leaves them uninitialised)."""
    from geographconv_amd import ops
    n, F = a.shape
    if dtype == 'f32':
        ld = ld or ops.pad4(F)
        t = torch.zeros((n, ld), dtype=torch.float32, device=dev)
    else:
        ld = ld or ops.bf16_ld(F)
        t = torch.zeros((n, ld), dtype=torch.bfloat16, device=dev)
    if junk:
        t[:, ops.pad4(F):] = float('nan')
    t[:, :F] = torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    return (ops.DMat if dtype == 'f32' else ops.HMat)(n, F, t=t)


def _f64(m):
    return m.t[:, :m.F].double().cpu().numpy()


def _vec(v, dev):
    return None if v is None else torch.from_numpy(np.pad(v, (0, -len(v) % 4))).to(dev)


def _problem(dev, M, K, N, dtype, bias, seed, act='silu', **kw):
    X, Wg, Wu = _rand((M, K), seed), _rand((K, N), seed + 1, 1 / np.sqrt(max(K, 1))), _rand((K, N), seed + 2, 1 / np.sqrt(max(K, 1)))
    bg, bu = (_rand((N,), seed + 3, 0.3), _rand((N,), seed + 4, 0.3)) if bias else (None, None)
    d = dict(X=_mat(X, dev, dtype, **kw), Wg=_mat(Wg, dev, dtype, **kw), Wu=_mat(Wu, dev, dtype, **kw), bg=_vec(bg, dev), bu=_vec(bu, dev))
    r = {k: _f64(d[k]) for k in ('X', 'Wg', 'Wu')}
    r['bg'], r['bu'] = (None if bg is None else bg.astype(np.float64)), (None if bu is None else bu.astype(np.float64))
    return d, r


def _forward_bounds(r, name, dtype):
    H, G, U = R.forward(r['X'], r['Wg'], r['Wu'], r['bg'], r['bu'], name)
    mg, mu = np.abs(r['X']) @ np.abs(r['Wg']), np.abs(r['X']) @ np.abs(r['Wu'])
    if r['bg'] is not None:
        mg, mu = mg + np.abs(r['bg']), mu + np.abs(r['bu'])
    v = np.abs(R.act(name, G)[0])
    h = 1.2 * np.abs(U) * ENV * mg + v * ENV * mu + EPS * v * np.abs(U) + EPS * np.abs(U) + 1e-30
    half = BF if dtype == 'bf16' else 2.0 ** -23
    return (H, h + half * np.abs(H)), (G, ENV * mg + half * np.abs(G) + 1e-30), (U, ENV * mu + half * np.abs(U) + 1e-30)


def _check(got, ref, what):
    want, bound = ref
    assert got.shape == want.shape and np.isfinite(got).all(), what
    bad = np.abs(got - want) > bound
    assert not bad.any(), "%s: %d of %d entries out of bounds, worst %.3g x" % (what, bad.sum(), bad.size, (np.abs(got - want) / bound).max())


FORWARD = [(1, 1, 1), (1, 300, 300), (1, 1024, 513), (2, 64, 32), (3, 33, 65), (7, 300, 930), (8, 129, 256), (9, 40, 7), (17, 1000, 31), (31, 2048, 40),
           (33, 7, 300), (64, 512, 96), (65, 100, 129), (128, 128, 128), (129, 300, 600), (200, 930, 517), (257, 65, 320), (700, 96, 161), (4500, 300, 300),
           (1000, 640, 1300), (16400, 300, 300), (16385, 600, 257), (17001, 40, 640), (16384, 200, 129)]


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('M,K,N', FORWARD)
def test_forward(dev, M, K, N, dtype):
    from geographconv_amd import ops
    name = ['silu', 'gelu', 'sigmoid', 'tanh', 'relu', 'none'][(M + K + N) % 6]
    d, r = _problem(dev, M, K, N, dtype, (M + N) % 2 == 0, M + K + N)
    ref = _forward_bounds(r, name, dtype)
    H = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=R.ACTS[name])
    _check(_f64(H), ref[0], 'H %s' % name)
    pads = H.t[:, N:ops.pad4(N) if dtype == 'f32' else H.ld].float()
    assert (pads == 0).all()
    H2, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=R.ACTS[name], keep='full')
    _check(_f64(H2), ref[0], 'H with G, U kept')
    _check(_f64(kept.G), ref[1], 'G')
    _check(_f64(kept.U), ref[2], 'U')
    H3, k8 = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=R.ACTS[name], keep='mx8')
    _check(_f64(H3), ref[0], 'H with checkpoints kept')
    for q, (want, bound) in ((k8.G, ref[1]), (k8.U, ref[2])):
        codes, scales, _ = R.mx8(want)
        got = _f64(ops.mx8_unpack(q))
        s = 2.0 ** (np.repeat(q.scales.cpu().numpy().astype(np.float64), 32, axis=1)[:, :N] - 127)
        half = np.maximum(2.0 ** -4 * (np.abs(want) + bound), 2.0 ** -10 * s)
        out16 = BF * np.abs(want) if dtype == 'bf16' else 0
        _check(got, (want, half * (1 + 1e-6) + bound + out16), 'checkpoint')
        if dtype == 'f32' and M < 16384:                 # ... and they are the codes of the very values the other form keeps (one kernel forms both)
            p = ops.mx8_pack(kept.G if q is k8.G else kept.U)
            assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)


@pytest.mark.parametrize('name', list(R.ACTS))
@pytest.mark.parametrize('M', [5, 300])
@pytest.mark.parametrize('precision', ['f32', 'bf16x3'])
def test_every_activation_in_both_fp32_precisions(dev, name, M, precision):
    from geographconv_amd import ops
    K, N = 70, 100
    d, r = _problem(dev, M, K, N, 'f32', True, 5)
    ref = _forward_bounds(r, name, 'f32')
    H, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=R.ACTS[name], keep='full', precision=precision)
    _check(_f64(H), ref[0], 'H')
    _check(_f64(kept.G), ref[1], 'G')
    dH = _mat(_rand((M, N), 8, 1e-3), dev, 'f32')
    _check_bwd(dev, d, r, dH, kept, name, 'f32', precision=precision)


def test_saturated_gates(dev):
    """Pre-activations from -200 to 200: no overflow on the way, the limits of each activation and derivative."""
    from geographconv_amd import ops
    g = np.concatenate([np.linspace(-200, 200, 64), [0, -0.0, 88.5, -88.5, 1e4, -1e4]]).astype(np.float32)
    N = len(g)
    X, Wg, Wu = np.ones((40, 1), np.float32), g[None, :].copy(), np.ones((1, N), np.float32)
    for name, code in R.ACTS.items():
        H, kept = ops.gated_dense(_mat(X, dev, 'f32'), _mat(Wg, dev, 'f32'), _mat(Wu, dev, 'f32'), act=code, keep='full')
        with np.errstate(over='ignore'):
            v, s = R.act(name, g.astype(np.float64))
        _check(_f64(H), (np.tile(v, (40, 1)), np.tile(EPS * np.abs(v) + EPS, (40, 1))), name)
        dX, dWg, dWu, _, _ = ops.gated_dense_bwd(_mat(np.ones((40, N), np.float32), dev, 'f32'), _mat(X, dev, 'f32'), _mat(Wg, dev, 'f32'),
                                                 _mat(Wu, dev, 'f32'), kept, act=code)
        _check(_f64(dWg) / 40, (s[None, :], EPS * (2 + np.abs(s[None, :]))), name + "'")


BACKWARD = [(1, 1, 1), (1, 300, 300), (2, 33, 65), (5, 64, 64), (31, 129, 40), (64, 300, 33), (130, 40, 300), (300, 257, 129), (1000, 300, 930), (5000, 96, 161),
            (4200, 300, 300), (700, 1100, 200), (16390, 300, 200), (16385, 129, 300), (16384, 192, 65), (17000, 400, 70)]


def _check_bwd(dev, d, r, dH, kept, name, dtype, X=None, precision=None, need_dx=True, bias=True):
    from geographconv_amd import ops
    X = d['X'] if X is None else X
    read = lambda m: _f64(ops.mx8_unpack(m)) if isinstance(m, ops.MX8Mat) else _f64(m)          # (mx8_unpack has its own tests)
    x, G, U, g = read(X), read(kept.G), read(kept.U), _f64(dH)
    dG, dU = R.gate_grads(g, G, U, name)
    eg, eu = EPS * (1 + np.abs(G)) * np.abs(g * U) + 1e-37, EPS * (1 + np.abs(G)) * np.abs(g) + 1e-37
    rnd = BF if dtype == 'bf16' else 0.0
    half = BF if dtype == 'bf16' else 2.0 ** -23
    wg, wu = np.abs(r['Wg']), np.abs(r['Wu'])
    res = ops.gated_dense_bwd(dH, X, d['Wg'], d['Wu'], kept, act=R.ACTS[name], bias=bias, need_input_grad=need_dx, precision=precision)
    if need_dx:
        dx = dG @ r['Wg'].T + dU @ r['Wu'].T
        mag = np.abs(dG) @ wg.T + np.abs(dU) @ wu.T
        _check(_f64(res[0]), (dx, (ENV + rnd) * mag + 2 * (eg @ wg.T + eu @ wu.T) + half * np.abs(dx) + 1e-30), 'dX')
    else:
        assert res[0] is None
    ax = np.abs(x).T
    for m, dd, e, what in ((res[1], dG, eg, 'dWg'), (res[2], dU, eu, 'dWu')):
        want = x.T @ dd
        _check(_f64(m), (want, (ENV + rnd) * (ax @ np.abs(dd)) + 2 * (ax @ e) + half * np.abs(want) + 1e-30), what)
    if bias:
        for v, dd, e, what in ((res[3], dG, eg, 'dbg'), (res[4], dU, eu, 'dbu')):
            _check(v[:dd.shape[1]].double().cpu().numpy(), (dd.sum(0), 128 * 2.0 ** -24 * np.abs(dd).sum(0) + e.sum(0) + 1e-30), what)
    return res


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('M,K,N', BACKWARD)
def test_backward(dev, M, K, N, dtype):
    from geographconv_amd import ops
    name = ['gelu', 'tanh', 'silu', 'sigmoid', 'relu', 'none'][(M + K + N) % 6]
    d, r = _problem(dev, M, K, N, dtype, False, M + 3 * K + N)
    kept = ops.GatedTape(_mat(_rand((M, N), 21), dev, dtype), _mat(_rand((M, N), 22), dev, dtype))
    dH = _mat(_rand((M, N), 23, 1e-3), dev, dtype)
    _check_bwd(dev, d, r, dH, kept, name, dtype)
    k8 = ops.GatedTape(ops.mx8_pack(kept.G), ops.mx8_pack(kept.U))
    x8 = ops.mx8_pack(d['X'])
    _check_bwd(dev, d, r, dH, k8, name, dtype, X=x8)
    _check_bwd(dev, d, r, dH, k8, name, dtype, need_dx=False, bias=False)
    if dtype == 'f32':
        _check_bwd(dev, d, r, dH, k8, name, dtype, X=x8, precision='f32')


def test_bf16_products_of_fp32_matrices(dev):
    """precision='bf16': operands rounded to bf16 (2^-8 each), accumulation fp32."""
    from geographconv_amd import ops
    M, K, N = 300, 130, 90
    d, r = _problem(dev, M, K, N, 'f32', True, 3)
    H, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=ops.ACT_SILU, keep='full', precision='bf16')
    mg = np.abs(r['X']) @ np.abs(r['Wg'])
    _, G, _ = R.forward(r['X'], r['Wg'], r['Wu'], r['bg'], r['bu'], 'silu')
    _check(_f64(kept.G), (G, (2 * BF + BF * BF + ENV) * mg + 1e-6), 'G')
    dH = _mat(_rand((M, N), 9), dev, 'f32')
    res = ops.gated_dense_bwd(dH, d['X'], d['Wg'], d['Wu'], kept, act=ops.ACT_SILU, precision='bf16')
    dG, dU = R.gate_grads(_f64(dH), _f64(kept.G), _f64(kept.U), 'silu')
    _check(_f64(res[1]), (r['X'].T @ dG, 3 * BF * (np.abs(r['X']).T @ np.abs(dG)) + 1e-5), 'dWg')


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_pitches_junk_pads_and_neighbouring_rows(dev, dtype):
    """Wider pitches with NaN behind roundup4(F), row views of a larger matrix, given outputs whose other rows stay as they were."""
    from geographconv_amd import ops
    M, K, N = 150, 70, 90
    ld = dict(f32=160, bf16=132)[dtype]
    d, r = _problem(dev, M, K, N, dtype, True, 12, ld=ld, junk=True)
    kind = ops.DMat if dtype == 'f32' else ops.HMat
    big = torch.full((M + 8, ld), 7.0, dtype=torch.float32 if dtype == 'f32' else torch.bfloat16, device=dev)
    out = kind(M + 8, N, t=big).rows(4, M + 4)
    H, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=ops.ACT_GELU, keep='full', out=out)
    _check(_f64(H), _forward_bounds(r, 'gelu', dtype)[0], 'H')
    assert (big[:4] == 7).all() and (big[M + 4:] == 7).all()
    dH = _mat(_rand((M, N), 14), dev, dtype, ld=ld, junk=True)
    _check_bwd(dev, d, r, dH, kept, 'gelu', dtype)
    d2, r2 = _problem(dev, M + 8, K, N, dtype, True, 12)
    d2['X'] = d2['X'].rows(3, M + 3)                      # (a view: its base lies inside a larger matrix)
    r2['X'] = r2['X'][3:M + 3]
    _check(_f64(ops.gated_dense(d2['X'], d2['Wg'], d2['Wu'], d2['bg'], d2['bu'], act=ops.ACT_SILU)), _forward_bounds(r2, 'silu', dtype)[0], 'view')
    _check(_f64(ops.gated_dense(d['X'], d['Wg'], d['Wu'], None, d['bu'], act=ops.ACT_SILU)),
           _forward_bounds(dict(r, bg=np.zeros(N)), 'silu', dtype)[0], 'one bias')


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('M', [9, 200, 16400])
def test_a_row_that_is_not_finite_stays_alone(dev, M, dtype):
    """An infinity or a NaN in a row of X reaches that row of H, G and U and no other; checkpoint blocks of the other rows are untouched too."""
    from geographconv_amd import ops
    d, _ = _problem(dev, M, 70, 100, dtype, True, 6)
    args = (d['Wg'], d['Wu'], d['bg'], d['bu'])
    want, kept = ops.gated_dense(d['X'], *args, act=ops.ACT_SILU, keep='full')
    want8, kept8 = ops.gated_dense(d['X'], *args, act=ops.ACT_SILU, keep='mx8')
    bad = [3, 8]
    d['X'].t[3, 5] = float('inf')
    d['X'].t[8, 69] = float('nan')
    got, gk = ops.gated_dense(d['X'], *args, act=ops.ACT_SILU, keep='full')
    got8, gk8 = ops.gated_dense(d['X'], *args, act=ops.ACT_SILU, keep='mx8')
    ok = torch.ones(M, dtype=torch.bool, device=dev)
    ok[bad] = False
    for a, b in ((want.t, got.t), (kept.G.t, gk.G.t), (kept.U.t, gk.U.t), (want8.t, got8.t), (kept8.G.codes, gk8.G.codes), (kept8.U.scales, gk8.U.scales)):
        assert torch.equal(a[ok], b[ok])
    assert not torch.isfinite(got.t[bad, :100].float()).any() and torch.isnan(got.t[8, :100].float()).all()
    assert not torch.isfinite(ops.mx8_unpack(gk8.G).t[bad, :100].float()).any()


def test_outputs_that_overlap_operands_are_refused(dev):
    from geographconv_amd import ops
    d, _ = _problem(dev, 20, 32, 32, 'f32', True, 1)
    _, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], keep='full')
    dH = _mat(_rand((20, 32), 2), dev, 'f32')
    for call in (lambda: ops.gated_dense(d['X'], d['Wg'], d['Wu'], out=d['X']),
                 lambda: ops.gated_dense_bwd(dH, d['X'], d['Wg'], d['Wu'], kept, dX=d['X']),
                 lambda: ops.gated_dense_bwd(dH, d['X'], d['Wg'], d['Wu'], kept, dWg=d['Wg'], dWu=_mat(_rand((32, 32), 3), dev, 'f32'))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_empty_sizes(dev, dtype):
    from geographconv_amd import ops
    kind = ops.DMat if dtype == 'f32' else ops.HMat
    tdt = torch.float32 if dtype == 'f32' else torch.bfloat16

    def z(n, F, v=0.0):
        return kind(n, F, t=torch.full((n, max(4, ops.pad4(F))), v, dtype=tdt, device=dev))
    H = ops.gated_dense(z(0, 8), z(8, 12), z(8, 12))
    assert H.n == 0 and H.F == 12
    dX, dWg, dWu, dbg, dbu = ops.gated_dense_bwd(z(0, 12), z(0, 8), z(8, 12), z(8, 12), ops.GatedTape(z(0, 12), z(0, 12)), dWg=z(8, 12, 3.0), dWu=z(8, 12, 3.0),
                                                 bias=True)
    assert dX.n == 0 and all((t == 0).all() for t in (dWg.t, dWu.t, dbg, dbu))
    x8 = ops.mx8_pack(z(0, 40))
    assert ops.mx8_unpack(x8).n == 0
    assert (ops.mx8_weight_grad(x8, z(0, 12), out=z(40, 12, 5.0)).t == 0).all()
    for n in (5, 40):                                     # no inputs: the biases alone
        H = ops.gated_dense(z(n, 0), z(0, 12), z(0, 12), bg=torch.full((12,), 2.0, device=dev), bu=torch.full((12,), 3.0, device=dev), act=ops.ACT_RELU)
        assert (H.t[:, :12] == 6).all()
    dX, dWg, _, dbg, dbu = ops.gated_dense_bwd(z(40, 12, 2.0), z(40, 0), z(0, 12), z(0, 12), ops.GatedTape(z(40, 12, 3.0), z(40, 12, 5.0)), act=ops.ACT_NONE, bias=True)
    assert dX.F == 0 and dWg.n == 0 and (dbg[:12] == 40 * 10).all() and (dbu[:12] == 40 * 6).all()


def _specials(n, F, seed):
    r = np.random.RandomState(seed)
    x = (r.randn(n, F) * 10.0 ** r.uniform(-6, 4, size=(n, 1))).astype(np.float32)
    x[0] = 0
    if n > 6:
        x[1, :5] = [448, 17, -17, 19, 2.0 ** -10]
        x[2, :3] = [np.inf, 1, 2]
        x[3, F // 2] = np.nan
        x[4] *= 2.0 ** -100
        x[5] = 2.0 ** -140
        x[6, 0] = 3e38
    return x


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('n,F', [(1, 1), (1, 32), (9, 33), (40, 300), (65, 31), (130, 64), (33, 1000), (2000, 600)])
def test_checkpoint_format(dev, n, F, dtype):
    from geographconv_amd import ops
    m = _mat(_specials(n, F, n + F), dev, dtype, junk=True, ld=(F + 35) // 32 * 32)
    q = ops.mx8_pack(m)
    with np.errstate(invalid='ignore'):
        codes, scales, values = R.mx8(_f64(m))
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    got = q.codes.cpu().numpy()
    assert np.array_equal(got & 0x7f, codes & 0x7f)
    assert np.array_equal(got[(codes & 0x7f) != 0], codes[(codes & 0x7f) != 0])            # (a zero's sign bit stands for nothing)
    back = ops.mx8_unpack(q)
    # (a value below 2^-133 is no bf16 number)
    tiny = np.abs(values) < 2.0 ** -126
    b = _f64(back)
    assert np.array_equal(b[~tiny], values[~tiny], equal_nan=True)
    if dtype == 'f32':
        assert np.array_equal(b[tiny], values[tiny])
    assert (back.t[:, F:] == 0).all()
    again = ops.mx8_pack(back)                            # what a checkpoint stands for is kept without a further change
    ok = np.repeat(scales != 255, 32, axis=1)[:, :F] & ~tiny
    assert np.array_equal(_f64(ops.mx8_unpack(again))[ok], values[ok])


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('M,K,N', [(1, 1, 1), (3, 33, 5), (40, 300, 129), (129, 64, 64), (1000, 300, 256), (5000, 200, 300), (300, 700, 1000), (16500, 300, 256), (20001, 33, 129), (16384, 320, 700), (100, 900, 700), (2000, 640, 1300), (513, 2048, 40)])
def test_weight_gradient_from_a_checkpoint(dev, M, K, N, dtype):
    from geographconv_amd import ops
    x8 = ops.mx8_pack(_mat(_rand((M, K), 1), dev, dtype))
    dZ = _mat(_rand((M, N), 2, 1e-2), dev, dtype)
    x, dz = _f64(ops.mx8_unpack(x8)), _f64(dZ)
    want, mag = x.T @ dz, np.abs(x).T @ np.abs(dz)
    for precision in (['bf16x3', 'f32'] if dtype == 'f32' else [None]):
        out = ops.mx8_weight_grad(x8, dZ, precision=precision)
        _check(_f64(out), (want, ENV * mag + (BF if dtype == 'bf16' else 2.0 ** -23) * np.abs(want) + 1e-30), 'dW')


def test_a_wide_range_of_magnitudes(dev):
    """fp32 values over 12 decades: the three terms of every value are exact at every exponent."""
    from geographconv_amd import ops
    M, K, N = 200, 96, 70
    rs = np.random.RandomState(4)
    X = (rs.randn(M, K) * 10.0 ** rs.uniform(-9, 3, size=(M, K))).astype(np.float32)
    d, r = _problem(dev, M, K, N, 'f32', False, 5)
    d['X'] = _mat(X, dev, 'f32')
    r['X'] = X.astype(np.float64)
    H, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], act=ops.ACT_NONE, keep='full')
    _check(_f64(kept.G), _forward_bounds(r, 'none', 'f32')[1], 'G')
    dH = _mat((rs.randn(M, N) * 10.0 ** rs.uniform(-9, 3, size=(M, N))).astype(np.float32), dev, 'f32')
    _check_bwd(dev, d, r, dH, kept, 'none', 'f32')


def test_gradients_against_differences(dev):
    """The directional derivative of sum(H * C) by central differences of the 64-bit forward, against the kernels' gradients."""
    from geographconv_amd import ops
    M, K, N = 37, 50, 44
    for name in ('silu', 'gelu', 'sigmoid', 'tanh', 'none'):
        d, r = _problem(dev, M, K, N, 'f32', True, 31)
        C = _rand((M, N), 40)
        _, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=R.ACTS[name], keep='full')
        g = ops.gated_dense_bwd(_mat(C, dev, 'f32'), d['X'], d['Wg'], d['Wu'], kept, act=R.ACTS[name], bias=True)
        grads = dict(X=_f64(g[0]), Wg=_f64(g[1]), Wu=_f64(g[2]), bg=g[3][:N].double().cpu().numpy(), bu=g[4][:N].double().cpu().numpy())
        for key, grad in grads.items():
            v = _rand(r[key].shape, 50).astype(np.float64)
            h = 1e-5
            f = [np.sum(C * R.forward(*[dict(r, **{key: r[key] + s * h * v})[k] for k in ('X', 'Wg', 'Wu', 'bg', 'bu')], name)[0]) for s in (1, -1)]
            num, ana = (f[0] - f[1]) / (2 * h), np.sum(grad * v)
            scale = np.sum(np.abs(grad * v))
            # differences: O(h^2) and 1e-16 |f| / h; the kernels: a few 1e-6 of the terms
            assert abs(num - ana) <= 1e-5 * scale + 1e-7, (name, key, num, ana)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_repeats_other_stream_and_graph(dev, dtype):
    """The same bits every time: again, on a side stream, and as a captured graph replayed between eager calls (two graphs share nothing)."""
    from geographconv_amd import ops
    M, K, N = 300, 200, 136
    d, r = _problem(dev, M, K, N, dtype, True, 77)
    dH = _mat(_rand((M, N), 78), dev, dtype)

    def step():
        H, kept = ops.gated_dense(d['X'], d['Wg'], d['Wu'], d['bg'], d['bu'], act=ops.ACT_SILU, keep='mx8')
        x8 = ops.mx8_pack(d['X'])
        out = ops.gated_dense_bwd(dH, x8, d['Wg'], d['Wu'], kept, act=ops.ACT_SILU, bias=True)
        dw = ops.mx8_weight_grad(x8, dH)
        return [H.t, out[0].t, out[1].t, out[2].t, out[3], out[4], dw.t]
    first = [t.clone() for t in step()]
    for t, u in zip(first, step()):
        assert torch.equal(t, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for t, u in zip(first, other):
        assert torch.equal(t, u)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    keep = d['X'].t.clone()
    for i in range(3):
        d['X'].t.copy_(keep * (i + 1))
        want = [t.clone() for t in step()]
        for g, outs in graphs:
            for t in outs:
                t.fill_(9)
            g.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            for a, b in zip(want, outs):
                assert torch.equal(a, b), i
