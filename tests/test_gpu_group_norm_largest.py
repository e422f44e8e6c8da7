"""Tensors just below 2 GiB: byte offsets up to 2^31, the first and the last image of every kernel family within their bounds
(tests/norm_bounds.py); codes, values and the weight gradient of the largest 8-bit copy."""
import numpy as np
import pytest

from oracle.keep8 import keep8_values
from tests import norm_bounds as nb
from tests.gpu_util import DevArr, say

pytestmark = pytest.mark.gpu


def part(api, ptr, at, n):
    """n floats from element `at` on."""
    out = np.empty(n, np.float32)
    api.memcpy_d2h(0, out, ptr + 4 * at)
    return out


@pytest.mark.parametrize('shape', [  # N, C, HW, groups, last: rows of channels; in registers, whole fours and ragged; split, last and first
    (131071, 4096, 1, 32, False), (8191, 64, 1024, 8, False), (8191, 65, 1007, 5, False), (2047, 256, 1024, 32, True),
    (2039, 257, 1023, 1, True), (4095, 2, 65537, 1, False)])
def test_group_norm(hip, shape):
    N, C, HW, G, last = shape
    per = C * HW
    n = N * per
    assert (1 << 29) - (1 << 22) < n < (1 << 29) - 1
    rs = np.random.RandomState(70)
    ga, be = rs.normal(1, 0.3, C).astype(np.float32), rs.normal(0, 0.3, C).astype(np.float32)
    GA, BE = DevArr(hip, ga), DevArr(hip, be)
    X, dY, Y, dX = (DevArr(hip, shape=(n,)) for _ in range(4))
    M, R, dG, dB = (DevArr(hip, shape=(k,), fill=np.nan) for k in (N * G, N * G, C, C))
    X8 = DevArr(hip, shape=((hip.bytes8(n) + 3) // 4,))
    hip.random_uniform(0, X.ptr, n, 71, -1.5, 2.0)
    # the channels' sums: dy is 0 but for the first and the last image
    hip.fill_f32(0, dY.ptr, 0.0, n)
    ends = [0, N - 1]
    dy = rs.normal(0, 1, (2, per)).astype(np.float32)
    for k, i in enumerate(ends):
        hip.memcpy_h2d(0, dY.ptr + 4 * i * per, dy[k])
    d = hip.group_norm_desc(N, C, HW, G, last, 2, 0.0, 1e-5)
    for kept in (False, True):
        say(f'largest group_norm {shape} kept={kept}')
        hip.fill_f32(0, Y.ptr, np.nan, n)
        hip.fill_f32(0, dX.ptr, np.nan, n)
        hip.group_norm_fwd(0, d, X.ptr, GA.ptr, BE.ptr, Y.ptr, M.ptr, R.ptr, X8.ptr if kept else None)
        hip.group_norm_bwd(0, d, None if kept else X.ptr, X8.ptr if kept else None, GA.ptr, BE.ptr, M.ptr, R.ptr, dY.ptr, dX.ptr, dG.ptr, dB.ptr)
        m, r = M.get().reshape(N, G), R.get().reshape(N, G)
        assert np.isfinite(m).all() and np.isfinite(r).all()
        sums = [0, 0, 0, 0]
        for k, i in enumerate(ends):
            # whole blocks of the copy around the image: blocks do not stop at its ends
            low, high = i * per // 32 * 32, min(n, -(-(i + 1) * per // 32) * 32)
            wide = part(hip, X.ptr, low, high - low)
            x = wide[i * per - low:][:per]
            mean, rstd, e_mean, e_rstd = nb.statistics(x, 1, C, HW, G, last, 1e-5)
            assert (np.abs(m[i] - mean) <= e_mean).all() and (np.abs(r[i] - rstd) <= e_rstd).all()
            y, e = nb.Pass(x, ga, be, m[i], r[i], 1, C, HW, G, last, 'silu', 0.0).forward()
            assert (np.abs(part(hip, Y.ptr, i * per, per) - y.reshape(-1)) <= e.reshape(-1)).all(), ('y', i)
            xs = keep8_values(wide)[i * per - low:][:per] if kept else x
            (dx, dg, db), (ex, eg, eb) = nb.Pass(xs, ga, be, m[i], r[i], 1, C, HW, G, last, 'silu', 0.0).backward(dy[k])
            assert (np.abs(part(hip, dX.ptr, i * per, per) - dx.reshape(-1)) <= ex.reshape(-1)).all(), ('dx', i)
            sums = [a + b for a, b in zip(sums, (dg, db, eg, eb))]
        dg, db, eg, eb = sums      # one more addition than in either image: part of H
        assert nb.telling([dg, db], [eg, eb]) == [True, True]
        assert (np.abs(dG.get() - dg) <= eg).all() and (np.abs(dB.get() - db) <= eb).all()
        # in between: gradients of zero
        mid = part(hip, dX.ptr, (N // 2) * per, min(per, 1 << 20))
        assert (mid == 0).all()


def test_copy_and_weight_gradient(hip):
    rows, K, M = 131071, 4096, 8
    n = rows * K
    say(f'largest copy, n={n}')
    X, B = DevArr(hip, shape=(n,)), DevArr(hip, shape=(n,), fill=np.nan)
    X8 = DevArr(hip, shape=((hip.bytes8(n) + 3) // 4,))
    hip.random_uniform(0, X.ptr, n, 72, -2.0, 2.0)
    hip.encode8(0, n, X.ptr, X8.ptr)
    hip.decode8(0, n, X8.ptr, B.ptr)
    for at in (0, n // 64 * 32, n - (1 << 20)):
        assert np.array_equal(part(hip, B.ptr, at, 1 << 20), keep8_values(part(hip, X.ptr, at, 1 << 20)))
    del B
    say('largest copy, weight gradient')
    rs = np.random.RandomState(73)
    codes = rs.randint(-3, 4, (rows, K), dtype=np.int8)
    hip.memcpy_h2d(0, X8.ptr, codes)
    hip.memcpy_h2d(0, X8.ptr + n, np.full(n // 32, 127, np.uint8))       # steps of 1
    dy = rs.randint(-4, 5, (rows, M)).astype(np.float32)
    dY, dW = DevArr(hip, dy), DevArr(hip, shape=(K, M), fill=np.nan)
    hip.gemm_wgrad8(0, 1, rows, K, M, X8.ptr, dY.ptr, dW.ptr)
    ref = np.zeros((K, M))
    for i in range(0, rows, 8192):       # whole numbers: each chunk below 2^24, exact in fp32
        ref += codes[i:i + 8192].astype(np.float32).T @ dy[i:i + 8192]
    assert np.array_equal(dW.get(), ref)
