"""What the tape of a network with 8-bit checkpoints holds (run on the MI355X: pytest -m gpu)."""
import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    from geographconv_amd import ops
    ops.require_gpu()
    return torch.device("cuda:0")


def _held(dev, n, F, hidden, checkpoint, linear_below):
    """-> (bytes on the device that the tape of one forward holds, its result's included; the gradients of one backward)"""
    from geographconv_amd import gcnmodel as M, ops
    from geographconv_amd.nn import layers as L, nonlinearities as NL
    np.random.seed(2)
    l_in = L.InputLayer((None, F))
    l = L.DenseLayer(l_in, F, nonlinearity=None if linear_below else NL.tanh)
    for h in hidden:
        l = M.gated_dense_block(l, h, checkpoint=checkpoint)
    params = L.get_all_params(l)
    store = L.ParamStore(params, dev)
    rs = np.random.RandomState(n)
    X, G = (ops.DMat.from_numpy(rs.randn(n, F).astype(np.float32), dev) for _ in range(2))
    L.get_output(l, {l_in: X}, tape={})                   # (what the library allocates once)
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(dev)
    tape = {}
    y = L.get_output(l, {l_in: X}, tape=tape)
    gc.collect()
    held = torch.cuda.memory_allocated(dev) - before
    L.backward(l, G, tape)
    return held, [store.read_grad(p) for p in params]


@pytest.mark.parametrize('linear_below', [False, True])
def test_a_checkpointed_network_holds_codes(dev, linear_below):
    """Blocks of F inputs and h hidden units: x, G, U and the hidden layer's output in 8 bits (33 / 32 bytes a value), the result, and the output
    of the tanh layer below, which that layer's own backward reads.  A linear layer below holds nothing."""
    n, F, hidden = 4096, 64, (128, 256, 96)
    held, grads = _held(dev, n, F, hidden, 'mx8', linear_below)
    codes = sum(n * (F + 3 * h) * 33 // 32 for h in hidden)
    want = codes + n * F * 4 * (1 if linear_below else 2)
    assert want <= held <= want + 512 * 40, (held, want)       # (the allocator's rounding: 512 bytes an allocation)
    full, exact = _held(dev, n, F, hidden, None, linear_below)
    assert held < 0.4 * full
    for a, b in zip(grads, exact):
        # (a checkpointed value is off by 2^-4 of itself at most, through up to four of them in a row)
        assert np.linalg.norm(a - b) <= 2.0 ** -4 * 4 * np.linalg.norm(b)
