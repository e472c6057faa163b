"""The gated dense block and the 8-bit checkpoints where the sizes, types and values of test_gated_gpu.py do not reach (run on the MI355X:
pytest -m gpu).  Bounds: as derived there (ENV * sum|a.b| for a product, half a step for a stored result); what is added is stated at each test."""
import numpy as np
import pytest

from . import gated_reference as R
from .test_gated_gpu import BF, ENV, EPS, _check, _f64, _mat, _problem, _rand

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
