"""What the gated dense block and the 8-bit checkpoints refuse, and the containers (no GPU: every call here is turned down on the host)."""
import ctypes as C

import numpy as np
import pytest
import torch

from geographconv_amd import _ffi, build, ops

from . import gated_reference as R

CPU = torch.device('cpu')


@pytest.fixture(scope='module')
def lib():
    build.build_library()
    return _ffi.lib()


def D(n, F, ld=None):
    return ops.DMat(n, F, CPU, ld=ld)


def Hm(n, F):
    return ops.HMat(n, F, t=torch.zeros(n, ops.bf16_ld(F), dtype=torch.bfloat16))


def Q(n, F, bf16=False):
    return ops.MX8Mat.empty(n, F, CPU, bf16)


def test_mx8mat_checks_its_parts():
    codes, scales = torch.zeros(5, 64, dtype=torch.uint8), torch.zeros(5, 2, dtype=torch.uint8)
    m = ops.MX8Mat(5, 40, codes, scales)
    assert m.ld == 64 and m.nbytes == 5 * 66
    for c, s, F in ((codes[:, ::2], scales, 20), (codes.float(), scales, 40), (codes, scales[:4], 40), (codes, scales, 65),
                    (torch.zeros(5, 40, dtype=torch.uint8), scales, 40), (codes, torch.zeros(5, 3, dtype=torch.uint8), 40)):
        with pytest.raises(ValueError):
            ops.MX8Mat(5, F, c, s)


def test_tape_is_of_one_kind():
    ops.GatedTape(D(3, 8), D(3, 8))
    for g, u in ((D(3, 8), Q(3, 8)), (D(3, 8), D(4, 8)), (D(3, 8), D(3, 4))):
        with pytest.raises(ValueError):
            ops.GatedTape(g, u)


@pytest.mark.parametrize('call', [
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 13)),
    lambda: ops.gated_dense(D(4, 8), D(9, 12), D(9, 12)),
    lambda: ops.gated_dense(D(4, 8), Hm(8, 12), Hm(8, 12)),
    lambda: ops.gated_dense(Hm(4, 8), Hm(8, 12), D(8, 12)),
    lambda: ops.gated_dense(Q(4, 8), D(8, 12), D(8, 12)),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), act=ops.ACT_SELU),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), act=99),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), keep='fp8'),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), precision='fp16'),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), bg=torch.zeros(11)),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), bu=torch.zeros(12, dtype=torch.float64)),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), bg=torch.zeros(24)[::2]),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), out=D(4, 8)),
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12), out=Hm(4, 12)),
    lambda: ops.gated_dense_bwd(D(4, 13), D(4, 8), D(8, 12), D(8, 12), ops.GatedTape(D(4, 12), D(4, 12))),
    lambda: ops.gated_dense_bwd(Hm(4, 12), D(4, 8), D(8, 12), D(8, 12), ops.GatedTape(D(4, 12), D(4, 12))),
    lambda: ops.gated_dense_bwd(D(4, 12), D(5, 8), D(8, 12), D(8, 12), ops.GatedTape(D(4, 12), D(4, 12))),
    lambda: ops.gated_dense_bwd(D(4, 12), Q(4, 8, True), D(8, 12), D(8, 12), ops.GatedTape(D(4, 12), D(4, 12))),
    lambda: ops.gated_dense_bwd(D(4, 12), D(4, 8), D(8, 12), D(8, 12), ops.GatedTape(D(5, 12), D(5, 12))),
    lambda: ops.gated_dense_bwd(D(4, 12), D(4, 8), D(8, 12), D(8, 12), ops.GatedTape(Q(4, 12, True), Q(4, 12, True))),
    lambda: ops.gated_dense_bwd(D(4, 12), D(4, 8), D(8, 12), D(8, 12), ops.GatedTape(D(4, 12), D(4, 12)), dWg=D(8, 12)),
    lambda: ops.gated_dense_bwd(D(4, 12), D(4, 8), D(8, 12), D(8, 12), ops.GatedTape(D(4, 12), D(4, 12)), dbg=torch.zeros(12)),
    lambda: ops.gated_dense_bwd(D(4, 12), D(4, 8), D(8, 12), D(8, 12), ops.GatedTape(D(4, 12), D(4, 12)), dX=D(4, 9)),
    lambda: ops.mx8_pack(Q(4, 8)),
    lambda: ops.mx8_pack(D(4, 8), out=Q(4, 8, True)),
    lambda: ops.mx8_pack(D(4, 8), out=Q(4, 9)),
    lambda: ops.mx8_unpack(D(4, 8)),
    lambda: ops.mx8_unpack(Q(4, 8), out=Hm(4, 8)),
    lambda: ops.mx8_weight_grad(Q(4, 8), D(5, 6)),
    lambda: ops.mx8_weight_grad(Q(4, 8), Hm(4, 6)),
    lambda: ops.mx8_weight_grad(D(4, 8), D(4, 6)),
    lambda: ops.mx8_weight_grad(Q(4, 8), Q(4, 6)),
    lambda: ops.mx8_weight_grad(Q(4, 8), D(4, 6), out=D(6, 8)),
])
def test_wrong_arguments_are_refused(call):
    with pytest.raises(ValueError):
        call()


def test_overlapping_outputs_are_refused():
    x, w = D(8, 8), D(8, 8)
    with pytest.raises(ValueError):
        ops._check_apart('x', [x], [w, x])
    big = D(20, 8)
    for outs, ins in (([big.rows(0, 8)], [big.rows(7, 15)]), ([x, x], [w]), ([big.rows(2, 4), big.rows(3, 5)], [])):
        with pytest.raises(ValueError):
            ops._check_apart('x', outs, ins)
    ops._check_apart('x', [big.rows(0, 8), None], [big.rows(8, 16), None, x])


@pytest.mark.parametrize('call', [
    lambda: ops.gated_dense(D(4, 8), D(8, 12), D(8, 12)),
    lambda: ops.gated_dense_bwd(D(4, 12), D(4, 8), D(8, 12), D(8, 12), ops.GatedTape(D(4, 12), D(4, 12))),
    lambda: ops.mx8_pack(D(4, 8)),
    lambda: ops.mx8_unpack(Q(4, 8)),
    lambda: ops.mx8_weight_grad(Q(4, 8), D(4, 6)),
])
def test_host_memory_is_refused(call):
    with pytest.raises(_ffi.GeoGcnError):
        call()


def _fwd(lib, **kw):
    """geogcn_gated_fwd with plausible (never dereferenced) addresses, some of them replaced -> return code, scratch asked for; without scratch a
    call of this many rows launches nothing."""
    a = dict(M=80, K=16, N=32, type=0, X=4096, ldx=16, Wg=8192, ldwg=32, Wu=12288, ldwu=32, bg=None, bu=None, act=5, H=16384, ldh=32, keep=0, G=None,
             ldg=0, Gs=None, U=None, ldu=0, Us=None, precision=1)
    a.update(kw)
    need = C.c_size_t(0)
    rc = lib.geogcn_gated_fwd(*a.values(), None, C.byref(need), None)
    return rc, need.value


def test_c_entry_refusals(lib):
    assert _fwd(lib)[0] == _ffi.E_WORKSPACE and _fwd(lib)[1] > 0
    for kw, rc in ((dict(M=-1), -2), (dict(N=1 << 21), -2), (dict(type=2), -4), (dict(act=3), -4), (dict(act=7), -4), (dict(keep=3), -4),
                   (dict(precision=3), -4), (dict(X=None), -1), (dict(Wu=None), -1), (dict(H=None), -1), (dict(X=4100), -3), (dict(ldx=18), -3),
                   (dict(ldx=12), -3), (dict(ldx=1 << 22), -2), (dict(ldh=28), -3), (dict(H=16392), -3), (dict(keep=1), -1), (dict(keep=2, G=64, ldg=32, U=64, ldu=32), -1),
                   (dict(keep=2, G=64, ldg=48, Gs=64, U=64, ldu=32, Us=64), -3), (dict(keep=1, type=1, ldh=64, G=64, ldg=32, U=64, ldu=64), -3)):
        got = _fwd(lib, **kw)[0]
        assert got == rc, (kw, got)
        assert lib.geogcn_last_error()
    assert lib.geogcn_gated_fwd(80, 16, 32, 0, 4096, 16, 8192, 32, 12288, 32, None, None, 5, 16384, 32, 0, None, 0, None, None, 0, None, 1, None, None,
                                None) == -1
    need = C.c_size_t(0)                                     # a workspace that is too small or badly placed is turned down before any launch
    args = (80, 16, 32, 0, 4096, 16, 8192, 32, 12288, 32, None, None, 5, 16384, 32, 0, None, 0, None, None, 0, None, 1)
    assert lib.geogcn_gated_fwd(*args, 256, C.byref(need), None) == _ffi.E_WORKSPACE and need.value == _fwd(lib)[1]
    need = C.c_size_t(1 << 30)
    assert lib.geogcn_gated_fwd(*args, 264, C.byref(need), None) == -3


def test_bwd_and_checkpoint_entry_refusals(lib):
    need = C.c_size_t(0)

    def bwd(**kw):
        a = dict(M=8, K=16, N=32, type=0, dH=4096, lddh=32, x_type=0, X=4096, ldx=16, Xs=None, Wg=4096, ldwg=32, Wu=4096, ldwu=32, kept_type=0, G=4096,
                 ldg=32, Gs=None, U=4096, ldu=32, Us=None, act=5, dX=4096, lddx=16, dWg=4096, lddwg=32, dWu=4096, lddwu=32, dbg=None, dbu=None,
                 precision=1)
        a.update(kw)
        return lib.geogcn_gated_bwd(*a.values(), None, C.byref(need), None)
    for kw in (dict(), dict(dX=None), dict(dWg=None, dWu=None), dict(dbg=4096, dbu=4096), dict(x_type=2, ldx=32, Xs=4096), dict(kept_type=2, Gs=4096, Us=4096)):
        need.value = 0
        assert bwd(**kw) == _ffi.E_WORKSPACE and need.value > 0, kw
    for kw, rc in ((dict(dWg=None), -1), (dict(dbu=4096), -1), (dict(x_type=1), -4), (dict(kept_type=1), -4), (dict(x_type=2, Xs=4096), -3),
                   (dict(kept_type=2, Gs=4096), -1), (dict(dbg=4100, dbu=4096), -3), (dict(lddx=12), -3), (dict(dH=None), -1), (dict(act=-1), -4),
                   (dict(K=-2), -2)):
        assert bwd(**kw) == rc, kw
    for args, rc in (((4, 8, 2, 4096, 8, 4096, 32, 4096), -4), ((4, 8, 0, 4096, 8, 4096, 8, 4096), -3), ((4, 8, 0, 4096, 6, 4096, 32, 4096), -3),
                     ((4, 8, 0, None, 8, 4096, 32, 4096), -1), ((-4, 8, 0, 4096, 8, 4096, 32, 4096), -2), ((4, 8, 0, 4100, 8, 4096, 32, 4096), -3)):
        assert lib.geogcn_mx8_pack(*args, None) == rc, args
    assert lib.geogcn_mx8_pack(0, 8, 0, None, 8, None, 32, None, None) == 0
    assert lib.geogcn_mx8_weight_grad(8, 16, 32, 0, 4096, 16, 4096, 4096, 32, 4096, 32, 1, None, C.byref(need), None) == -3
    assert lib.geogcn_mx8_weight_grad(8, 16, 32, 0, 4096, 32, None, 4096, 32, 4096, 32, 1, None, C.byref(need), None) == -1


def test_reference_format_by_hand():
    """The checker itself: a block's scale, ties, the subnormal end, signs, a block that is not finite."""
    x = np.zeros((3, 33))
    x[0, :6] = [448, 1.0, -17, 17.5, 2.0 ** -10, 3 * 2.0 ** -10]     # scale 1: 17 lies between 16 and 18 (tie to 16), 2^-10 half the last step
    x[0, 32] = 449                                                    # its own block: 449 > 448, so the scale is 2
    x[1, 3] = np.inf
    codes, scales, v = R.mx8(x)
    assert scales.tolist() == [[127, 128], [255, 1], [1, 1]]
    assert v[0, :6].tolist() == [448, 1, -16, 18, 0, 2.0 ** -8] and v[0, 32] == 448
    assert np.isnan(v[1, :32]).all() and v[1, 32] == 0 and (v[2] == 0).all()
    assert codes[0, 0] == 0x7e and codes[0, 1] == 0x38 and codes[0, 2] == 0x80 | 0x58
