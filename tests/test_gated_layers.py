"""Construction of the gated layer and block (no GPU)."""
import numpy as np
import pytest

from geographconv_amd import gcnmodel as M
from geographconv_amd.nn import layers as L
from geographconv_amd.nn import nonlinearities as NL


def test_parameters_and_shapes():
    np.random.seed(1)
    l_in = L.InputLayer((None, 20))
    g = L.GatedDenseLayer(l_in, 33, nonlinearity=NL.gelu)
    assert g.output_shape == (None, 33) and [p.shape for p in L.get_all_params(g)] == [(20, 33), (20, 33), (33,), (33,)]
    assert [p.shape for p in L.get_all_params(g, regularizable=True)] == [(20, 33), (20, 33)]
    block = M.gated_dense_block(l_in, checkpoint='mx8')
    assert block.output_shape == (None, 20) and L.count_params(block) == 2 * (20 * 40 + 40) + 40 * 20 + 20


@pytest.mark.parametrize('make', [
    lambda i: L.GatedDenseLayer(i, 8, nonlinearity=NL.softmax),
    lambda i: L.GatedDenseLayer(i, 8, nonlinearity=NL.selu),
    lambda i: L.GatedDenseLayer(i, 8, bg=None),
    lambda i: L.GatedDenseLayer(i, 8, checkpoint='fp8'),
    lambda i: L.DenseLayer(i, 8, checkpoint='int8'),
    lambda i: M.gated_dense_block(i, checkpoint=8),
])
def test_refusals(make):
    with pytest.raises(ValueError):
        make(L.InputLayer((None, 20)))


def test_gates_are_not_dense_activations():
    with pytest.raises(NotImplementedError):
        L.DenseLayer(L.InputLayer((None, 20)), 8, nonlinearity=NL.swish)._fused_act()
