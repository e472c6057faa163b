"""Which tile shape and split a product of the gated dense block runs on: the tables and the estimate of csrc/gated.hip (run_best), read from the
source and replayed, so that the sizes of test_gated_range_gpu.py can be shown to reach every entry (test infrastructure)."""
import os
import re

CUS = 256
SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'geographconv_amd', 'csrc', 'gated.hip')


def tables():
    """{'run_forward/fp32': [(rows, columns of a segment, k of a stage, stages, blocks a CU, eff), ...], ...}"""
    src = open(SOURCE).read()
    out = {}
    for fn in ('run_forward', 'run_input_grad', 'run_weight_grad'):
        body = src[src.index('int %s(' % fn):]
        body = body[:body.index('\n}\n')]
        for name, entries in re.findall(r'static const Shape (\w+)\[\] = \{(.*?)\};', body, re.S):
            found = re.findall(r'\{(\d+), (\d+), (\d+), (\d+), (\d+), ([0-9.]+), run_tiles<', entries)
            assert found and entries.count('run_tiles<') == len(found)
            out['%s/%s' % (fn, name)] = [tuple(int(v) for v in e[:5]) + (float(e[5]),) for e in found]
    return out


def cdiv(a, b):
    return -(-a // b)


def up(n, m):
    return cdiv(n, m) * m


def best(shapes, M, cols, K, kseg, nseg, terms):
    """-> (index of the entry, number of splits)"""
    pick = None
    for i, (bm, bns, bk, stages, per_cu, eff) in enumerate(shapes):
        n_mt, n_nt = cdiv(M, bm), cdiv(cols, bns)
        tiles, steps = n_mt * n_nt, max(1, kseg * cdiv(K, bk))
        want = 1
        while want == 1 or (want <= steps // 4 and tiles * want <= 2 * CUS):
            per = cdiv(steps, want)
            nsplit = cdiv(steps, per)
            R = cdiv(tiles * nsplit, CUS)
            turns = cdiv(R, per_cu)
            clk = max(R * bm * bns * nseg * (per * bk) * terms / (2048 * 0.7 * eff), turns * per * 1900 / (stages - 1)) + turns * 6000.0
            if nsplit > 1:
                clk += 2.0 * nsplit * M * n_nt * bns * nseg * 4 / 1500 + 16000
            if pick is None or clk < pick[0]:
                pick = (clk, i, nsplit)
            want += 1 if want < 8 else want // 4
    return pick[1:]


def _cols(F, bf16):
    return up(F, 64 if bf16 else 4)


def forward(t, M, K, N, dtype, precision='bf16x3', keep=None):
    """-> (table, entry, splits), None: not by tiles"""
    one = dtype == 'bf16' or precision == 'bf16'
    if M <= 16 and not (dtype == 'f32' and one):
        return None
    if not one and keep != 'mx8' and M >= (32768 if max(K, N) > 640 else 16384):
        return None
    name = 'run_forward/' + ('bf16' if one else 'fp32')
    cols = _cols(N, dtype == 'bf16')
    return (name,) + best(t[name], M, max(cols, up(N, 32)) if keep == 'mx8' else cols, K, 1, 2, 1 if one else 6)


def _library(M, K, N, dtype, precision):
    return dtype == 'f32' and precision == 'bf16x3' and M >= 16384 and 192 <= K <= 320 and N <= 1024


def input_grad(t, M, K, N, dtype, precision='bf16x3'):
    if _library(M, K, N, dtype, precision):
        return None
    terms = 1 if precision == 'bf16' else 2 if dtype == 'bf16' else 3
    name = 'run_input_grad/' + {1: 'bf16', 2: 'two', 3: 'fp32'}[terms]
    return (name,) + best(t[name], M, _cols(K, dtype == 'bf16'), N, 2, 1, {1: 1, 2: 2, 3: 6}[terms])


def weight_grads(t, M, K, N, dtype, precision='bf16x3', eight=False):
    if _library(M, K, N, dtype, precision):
        return None
    name = 'bf16' if precision == 'bf16' else 'two' if dtype == 'bf16' else 'mx8' if eight else 'fp32'
    name, terms = 'run_weight_grad/' + name, dict(bf16=1, two=2, mx8=3, fp32=6)[name]
    return (name,) + best(t[name], K, _cols(N, dtype == 'bf16'), M, 1, 2, terms)


def weight_grad(t, M, K, N, dtype, precision='bf16x3'):
    three = dtype == 'f32' and precision == 'bf16x3'
    if three and min(K, N) <= 640 and max(K, N) <= 2048:
        return None
    name = 'run_weight_grad/' + ('mx8_one' if three else 'bf16_one')
    return (name,) + best(t[name], K, _cols(N, dtype == 'bf16'), M, 1, 1, 3 if three else 1)


# (rows, inputs, units, type, precision): odd sizes that between them run every entry of the tables, with its reduction whole and split
FORWARD = [(M, K, N, 'f32', 'bf16x3') for M, K, N in ((6692, 47, 261), (799, 1941, 873), (11185, 35, 277), (3674, 2373, 275), (34, 31, 31), (37, 422, 31))]
FORWARD += [(M, K, N, dt, 'bf16') for M, K, N in ((286, 51, 5495), (33, 1902, 70), (19135, 42, 134), (60, 2291, 33), (781, 33, 4790), (6, 2793, 811),
                                                   (34, 31, 31), (37, 1446, 34)) for dt in ('f32', 'bf16')]
# ... and 8-bit X, G, U?
BACKWARD = [(M, K, N, 'f32', 'bf16x3', e) for M, K, N, e in ((17430, 398, 34, False), (2052, 153, 1317, False), (17078, 146, 37, True), (458, 1551, 1259, False),
                                                             (34, 31, 31, True), (32, 63, 198, False), (244, 30, 41, False), (47, 677, 5510, True),
                                                             (611, 713, 154, True), (457, 30, 37, True))]
BACKWARD += [(M, K, N, 'bf16', 'bf16x3', e) for M, K, N, e in ((17430, 398, 34, True), (1970, 2066, 1838, False), (17078, 146, 37, False), (1056, 1974, 2347, True),
                                                               (34, 31, 31, False), (37, 33, 393, True), (506, 30, 42, False), (67, 2783, 1414, False),
                                                               (999, 369, 46, True))]
BACKWARD += [(M, K, N, 'f32', 'bf16', e) for M, K, N, e in ((17430, 398, 34, True), (4139, 958, 3809, False), (17078, 146, 37, False), (1018, 1289, 5073, True),
                                                            (34, 31, 31, True), (51, 37, 671, False), (41, 262, 5487, True), (1872, 22, 4130, False),
                                                            (1339, 35, 39, True))]
BACKWARD += [(M, K, N, 'bf16', 'bf16', e) for M, K, N, e in ((600, 264, 1000, False), (4097, 520, 200, True))]
WEIGHT = [(47, 677, 5510, 'f32', 'bf16x3'), (1652, 1857, 2185, 'f32', 'bf16x3'), (40, 30, 2109, 'f32', 'bf16x3'), (633, 39, 2194, 'f32', 'bf16x3'),
          (34, 31, 31, 'f32', 'bf16'), (1692, 31, 31, 'f32', 'bf16'), (300, 64, 129, 'bf16', 'bf16x3'), (1000, 300, 256, 'f32', 'bf16')]
