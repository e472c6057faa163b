"""A network with gated blocks, trained through the layer API, against a 64-bit torch restatement (run on the MI355X: pytest -m gpu)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    from geographconv_amd import ops
    ops.require_gpu()
    return torch.device("cuda:0")


def _net(seed, checkpoint, classes=7, F=44, hidden=60):
    from geographconv_amd import gcnmodel as M
    from geographconv_amd.nn import layers as L, nonlinearities as NL
    np.random.seed(seed)
    l_in = L.InputLayer((None, F))
    l = L.DenseLayer(l_in, hidden, nonlinearity=NL.tanh)
    l = M.gated_dense_block(l, 90, nonlinearity=NL.swish, checkpoint=checkpoint)
    l = M.gated_dense_block(l, 50, nonlinearity=NL.gelu, checkpoint=checkpoint)
    return l_in, L.DenseLayer(l, classes, nonlinearity=NL.softmax)


def _step(dev, l_in, l_out, X, y, store, **kw):
    from geographconv_amd import ops
    from geographconv_amd.nn import layers as L
    tape = {}
    P = L.get_output(l_out, {l_in: X}, tape=tape, **kw)
    idx = torch.arange(X.n, dtype=torch.int32, device=dev)
    dl = ops.softmax_ce_bwd(P, idx, y)
    L.backward(l_out, L.PreAct(dl), tape, **kw)
    return P, tape


def _reference(values, X, y):
    """The same network in float64 on the CPU, gradients by autograd."""
    ps = [torch.tensor(v, dtype=torch.float64, requires_grad=True) for v in values]
    W, b = ps[0], ps[1]
    h = torch.tanh(X @ W + b)
    for k, act in ((2, torch.nn.functional.silu), (8, torch.nn.functional.gelu)):
        Wg, Wu, bg, bu, Wd, bd = ps[k:k + 6]
        h = (act(h @ Wg + bg) * (h @ Wu + bu)) @ Wd + bd + h
    logits = h @ ps[14] + ps[15]
    loss = torch.nn.functional.cross_entropy(logits, y)
    loss.backward()
    return torch.softmax(logits, 1).detach().numpy(), [p.grad.numpy() for p in ps]


@pytest.mark.parametrize('n', [40, 700])
@pytest.mark.parametrize('precision', ['bf16x3', 'f32'])
def test_network_gradients(dev, n, precision):
    from geographconv_amd import ops
    from geographconv_amd.nn import layers as L
    l_in, l_out = _net(3, None)
    params = L.get_all_params(l_out)
    store = L.ParamStore(params, dev)
    rs = np.random.RandomState(n)
    X, y = rs.randn(n, 44).astype(np.float32), rs.randint(0, 7, n)
    P, _ = _step(dev, l_in, l_out, ops.DMat.from_numpy(X, dev), torch.from_numpy(y.astype(np.int32)).to(dev), store, gemm_precision=precision)
    wantP, want = _reference([p.get_value() for p in params], torch.tensor(X, dtype=torch.float64), torch.tensor(y))
    # fp32 against 64 bits through six products of widths up to 90: a few 1e-6 of the largest entry each
    assert np.abs(P.numpy() - wantP).max() <= 2e-5
    for p, g in zip(params, want):
        got = store.read_grad(p)
        assert np.abs(got - g).max() <= 5e-5 * np.abs(g).max() + 1e-9, p.name


def test_checkpointed_layers_run_from_the_codes(dev):
    """checkpoint='mx8': the forward's bits are unchanged, the tape holds codes, and the gradients are those of the checkpointed values."""
    from geographconv_amd import ops
    from geographconv_amd.nn import layers as L, nonlinearities as NL
    rs = np.random.RandomState(8)
    n, F, N, C = 300, 44, 60, 20
    X = ops.DMat.from_numpy(rs.randn(n, F).astype(np.float32), dev)
    G = ops.DMat.from_numpy(rs.randn(n, C).astype(np.float32), dev)
    outs, grads = [], []
    for ck in (None, 'mx8'):
        np.random.seed(4)
        l_in = L.InputLayer((None, F))
        l1 = L.DenseLayer(l_in, F, nonlinearity=NL.tanh)
        l2 = L.GatedDenseLayer(l1, N, nonlinearity=NL.swish, checkpoint=ck)
        l3 = L.DenseLayer(l2, C, nonlinearity=None, checkpoint=ck)
        params = L.get_all_params(l3)
        store = L.ParamStore(params, dev)
        tape = {}
        y = L.get_output(l3, {l_in: X}, tape=tape)
        L.backward(l3, G, tape)
        outs.append(y.numpy())
        grads.append([store.read_grad(p) for p in params])
        if ck:
            assert all(isinstance(m, ops.MX8Mat) for m in (tape[l2]['x'], tape[l2]['kept'].G, tape[l2]['kept'].U, tape[l3]['x']))
            assert l1 not in tape['__values__'] and l2 not in tape['__values__']
            # the same by hand
            dh = ops.gemm(G, l3.W.data, transB=True)
            dW3 = ops.mx8_weight_grad(tape[l3]['x'], G)
            d1, dWg, dWu, dbg, dbu = ops.gated_dense_bwd(dh, tape[l2]['x'], l2.Wg.data, l2.Wu.data, tape[l2]['kept'], act=ops.ACT_SILU, bias=True)
            for got, want in ((l3.W.grad.t, dW3.t), (l2.Wg.grad.t, dWg.t), (l2.Wu.grad.t, dWu.t)):
                assert torch.equal(got[:, :want.shape[1]], want)
            assert torch.equal(l2.bg.grad[:N], dbg[:N]) and torch.equal(l2.bu.grad[:N], dbu[:N])
    assert np.array_equal(*outs)
    for a, b in zip(*grads):
        # every checkpointed value is off by 2^-4 of itself at most; the gradients of random data by less than that in the norm
        assert np.linalg.norm(a - b) <= 2.0 ** -4 * 2 * np.linalg.norm(a)


def test_a_graph_layer_refuses_a_checkpoint(dev):
    from geographconv_amd import gcnmodel as M, ops
    from geographconv_amd.nn import layers as L
    import scipy.sparse as sps
    l_in = L.InputLayer((None, 8))
    conv = M.ConvolutionDenseLayer2(l_in, num_units=8, checkpoint='mx8')
    L.ParamStore(L.get_all_params(conv), dev)
    A = ops.SparseOperand.from_scipy(sps.identity(16, format='csr', dtype=np.float32), dev)
    with pytest.raises(ValueError):
        L.get_output(conv, {l_in: ops.DMat.from_numpy(np.ones((16, 8)), dev)}, A=A, tape={})


def test_a_captured_step_replays_the_eager_one(dev):
    """A step of a checkpointed network captured into a graph and replayed between eager steps gives the eager gradients every time."""
    from geographconv_amd import ops
    from geographconv_amd.nn import layers as L
    l_in, l_out = _net(5, 'mx8')
    params = L.get_all_params(l_out)
    store = L.ParamStore(params, dev)
    rs = np.random.RandomState(1)
    X = ops.DMat.from_numpy(rs.randn(130, 44).astype(np.float32), dev)
    y = torch.from_numpy(rs.randint(0, 7, 130).astype(np.int32)).to(dev)
    _step(dev, l_in, l_out, X, y, store)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        P, _ = _step(dev, l_in, l_out, X, y, store)
    base = X.t.clone()
    for i in range(3):
        X.t.copy_(base * (1 + i))
        eager = _step(dev, l_in, l_out, X, y, store)[0].t.clone()
        want = store.g.clone()
        store.g.fill_(5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(P.t, eager)
        for p, a, b in ((p, store.read_grad(p), w) for p, w in zip(params, _split(store, want))):
            assert np.array_equal(a, b), (i, p.name)


def _split(store, flat):
    g, store.g = store.g.clone(), store.g
    store.g.copy_(flat)
    out = [store.read_grad(p) for p in store.params]
    store.g.copy_(g)
    return out
