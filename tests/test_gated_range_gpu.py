"""The gated dense block and the 8-bit checkpoints where the sizes, types and values of test_gated_gpu.py do not reach (run on the MI355X:
pytest -m gpu).  Bounds: as derived there (ENV * sum|a.b| for a product, half a step for a stored result); what is added is stated at each test."""
import numpy as np
import pytest

from . import gated_reference as R
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
