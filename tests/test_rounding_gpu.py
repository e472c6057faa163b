"""Where each sum of the update and of the gating mix is rounded: bit for bit against fp32 NumPy (run on the MI355X: pytest -m gpu)."""
import numpy as np
import pytest
import scipy.sparse as sps

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    from geographconv_amd import ops
    ops.require_gpu()
    return torch.device("cuda:0")


def test_adam_rounds_every_product_of_its_two_averages(dev):
    """m = b1 m + (1 - b1) g and v = b2 v + ((1 - b2) g) g, both products and the sum rounded each; the penalty's sum likewise."""
    from geographconv_amd import ops
    f = np.float32
    n = 40007
    rs = np.random.RandomState(0)
    p, m = rs.randn(n).astype(f), (rs.randn(n) * 0.1).astype(f)
    v = (m * m).astype(f)
    mask = (np.arange(n) % 3 != 0).astype(f)
    b1, b2, l1, l2 = f(0.9), f(0.999), f(1e-3), f(3e-4)
    tp, tm, tv, tr = (torch.from_numpy(a.copy()).to(dev) for a in (p, m, v, mask))
    for t in range(1, 4):
        g = (rs.randn(n) * 0.1).astype(f)
        tg = torch.from_numpy(g.copy()).to(dev)
        p = tp.cpu().numpy()
        ops.adam_step(tp, tg, tm, tv, tr, 2e-3, 0.9, 0.999, 1e-8, t, l1=float(l1), l2=float(l2))
        g = g + mask * (l1 * np.sign(p) + f(2) * l2 * p)             # (a mask of zeros and ones: its product is exact)
        m = b1 * m + (f(1) - b1) * g
        v = b2 * v + (f(1) - b2) * g * g
        for a, b, what in ((tg, g, 'g'), (tm, m, 'm'), (tv, v, 'v')):
            assert b.dtype == f and np.array_equal(a.cpu().numpy(), b), (what, t)


@pytest.mark.parametrize('F', [12, 64, 100, 300, 600])
def test_the_gating_mix_is_the_same_in_every_column_fused_or_not(dev, F):
    """T Hc + (1 - T) H in the product's epilogue and in its own pass: the same bits in every column, and they are those of one rounding of
    T Hc + r with r = (1 - T) H rounded before."""
    from geographconv_amd import ops
    n = 500
    rs = np.random.RandomState(F)
    A = ops.CSR(sps.random(n, n, 0.05, format='csr', random_state=1, dtype=np.float32), dev)
    B, T, H = (ops.DMat.from_numpy(a, dev) for a in (rs.randn(n, F), rs.rand(n, F), rs.randn(n, F)))
    bias = torch.from_numpy(rs.randn(ops.pad4(F)).astype(np.float32)).to(dev)
    Hc, fused = ops.spmm_highway(A, B, bias, T, H)
    assert np.array_equal(fused.numpy(), ops.highway_fwd(T, Hc, H).numpy())
    t, hc, h = T.numpy(), Hc.numpy(), H.numpy()
    r = (np.float32(1) - t) * h
    # (the product is exact in 64 bits; the sum of it and an fp32 number rounds there too, which can only move a result that lies between two fp32 numbers to
    # 2^-29 of their distance: such entries are left out)
    s = t.astype(np.float64) * hc + r
    one = s.astype(np.float32)
    gap = np.abs(np.spacing(one).astype(np.float64))
    clear = np.abs(np.abs(s - one) - gap / 2) > gap * 2.0 ** -20
    assert clear.mean() > 0.99 and np.array_equal(fused.numpy()[clear], one[clear])
