"""Calls of the gated dense block and the 8-bit checkpoints that are turned down on the host, and what their sources state (no GPU)."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch
from scipy.special import erfcx

from geographconv_amd import _ffi, build, ops

from . import gated_shapes as S
from .test_gated import D, Hm, Q


def _shared(n, F, kind):
    """-> a dense matrix and a checkpoint in one piece of memory: the matrix' last row holds the checkpoint's scales (or codes)"""
    w = (F + 31) // 32
    if kind == 'scales':
        ld = max(ops.pad4(F), (n * w + 3) // 4 * 4)
        raw = torch.zeros(n * ld * 4, dtype=torch.uint8)
        scales = raw[(n - 1) * ld * 4:][:n * w].view(n, w)
        codes = torch.zeros(n, 32 * w, dtype=torch.uint8)
    else:
        ld = max(ops.pad4(F), 8 * w * n)
        raw = torch.zeros(n * ld * 4, dtype=torch.uint8)
        codes = raw[(n - 1) * ld * 4:][:n * 32 * w].view(n, 32 * w)
        scales = torch.zeros(n, w, dtype=torch.uint8)
    return ops.DMat(n, F, t=raw.view(torch.float32).view(n, ld)), ops.MX8Mat(n, F, codes, scales)


@pytest.mark.parametrize('kind', ['codes', 'scales'])
def test_overlapping_outputs_of_the_checkpoint_calls_are_refused(kind):
    m, q = _shared(4, 40, kind)
    z = D(4, 40)
    for call in (lambda: ops.mx8_pack(m, out=q), lambda: ops.mx8_unpack(q, out=m)):
        with pytest.raises(ValueError, match='overlaps'):
            call()
    m, q = _shared(40, 40, kind)
    with pytest.raises(ValueError, match='overlaps'):
        ops.mx8_weight_grad(q, D(40, 40), out=m)
    with pytest.raises(ValueError, match='overlaps'):
        ops._check_apart('x', [m], [z, q])
    ops._check_apart('x', [D(40, 40)], [z, q, m])


def test_a_weight_gradient_over_its_own_operand_is_refused():
    for z, q in ((D(8, 8), Q(8, 8)), (Hm(8, 8), Q(8, 8, True))):
        with pytest.raises(ValueError, match='overlaps'):
            ops.mx8_weight_grad(q, z, out=z)
    big = D(20, 8)
    with pytest.raises(ValueError, match='overlaps'):
        ops.mx8_weight_grad(Q(8, 8), big.rows(0, 8), out=big.rows(7, 15))


def test_the_gpu_tests_run_every_tile_shape():
    """The sizes that test_gated_range_gpu.py compares reach every entry of csrc/gated.hip's tables, with the reduction whole and split."""
    t = S.tables()
    seen = {S.forward(t, *c) for c in S.FORWARD}
    seen |= {S.input_grad(t, *c[:5]) for c in S.BACKWARD} | {S.weight_grads(t, *c) for c in S.BACKWARD} | {S.weight_grad(t, *c) for c in S.WEIGHT}
    seen = {(s[0], s[1], s[2] > 1) for s in seen if s}
    want = {(name, i, split) for name, shapes in t.items() for i in range(len(shapes)) for split in (False, True)}
    assert seen == want, sorted(want - seen)


@pytest.fixture(scope='module')
def lib():
    build.build_library()
    return _ffi.lib()


def test_sizes_that_no_launch_holds_are_refused_before_any(lib):
    """2^31 rows (allowed by the checks of the single sizes) are more blocks of a tile than a launch has: refused when the scratch is asked for, not
    by the launch itself after others ran."""
    rows, need = 1 << 31, C.c_size_t(0)

    def fwd(M, type):
        return lib.geogcn_gated_fwd(M, 4, 4, type, 4096, 4, 4096, 4, 4096, 4, None, None, 5, 4096, 4, 0, None, 0, None, None, 0, None, 1, None, C.byref(need), None)

    def bwd(M, type):
        return lib.geogcn_gated_bwd(M, 4, 4, type, 4096, 4, type, 4096, 4, None, 4096, 4, 4096, 4, type, 4096, 4, None, 4096, 4, None, 5, 4096, 4, 4096, 4,
                                    4096, 4, None, None, 1, None, C.byref(need), None)
    for call in (fwd, bwd):
        for type in (0, 1):
            need.value = 0
            assert call(rows, type) == -2 and b'too large' in lib.geogcn_last_error(), (call, type)
            assert need.value == 0
    assert fwd(1 << 24, 0) == _ffi.E_WORKSPACE and bwd(1 << 24, 0) == _ffi.E_WORKSPACE


def test_the_normal_distributions_polynomial_has_the_error_it_states():
    """gate.h, normal_fast: R(t) against exp(z^2) erfc(z), z = |x| / sqrt 2, t = 1 / (1 + 0.3 |x|), with the committed coefficients."""
    src = open(os.path.join(os.path.dirname(S.SOURCE), 'gate.h')).read()
    k = [float(v.rstrip('f')) for v in re.search(r'k\[10\] = \{(.*?)\}', src).group(1).split(', ')]
    stated = float(re.search(r'ten terms t \.\. t\^10, largest error ([0-9.e-]+)', src).group(1))
    t = np.linspace(1e-6, 1, 1000001)
    error = np.abs(sum(c * t ** (i + 1) for i, c in enumerate(k)) - erfcx((1 / t - 1) / (0.3 * np.sqrt(2))))
    assert 0.9 * stated < error.max() <= stated
