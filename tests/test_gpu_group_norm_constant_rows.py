"""Rows of one repeated value: the sums of such values are rounded like any others, so the mean may miss the value by that much,
and rstd is then up to 1 / sqrt(eps).

With dm the bound of the mean's error (tests/norm_bounds.py: (H + 8 J) u |c|) every partial mean lies within dm of c, so that
the squared distances of values and partial means from the mean add up to at most (2 dm)^2 a value.  y is compared at the mean
and rstd that were stored; what is left of the value itself in y is at most dm rstd gamma."""
import numpy as np
import pytest

from tests import norm_bounds as nb
from tests.gpu_util import DevArr, say

pytestmark = pytest.mark.gpu
SHAPES = [(2, 6, 10, 3), (1, 8, 9000, 2), (5, 16, 1, 4), (3, 4, 1, 4), (2, 100, 36, 1), (1, 8, 70000, 2), (3, 64, 4097, 4), (4, 2500, 1, 1), (2, 9000, 1, 1)]


@pytest.mark.parametrize('value', [0.1, 1000.1, -3.3e-5, 12345.678, 0.0])
@pytest.mark.parametrize('last', [False, True])
def test_rows_of_one_value(hip, last, value):
    eps = 1e-5
    for N, C, HW, G in SHAPES:
        say(f'constant rows {N} {C} {HW} {G} last={last} value={value}')
        x = np.full((N, HW, C) if last else (N, C, HW), value, np.float32)
        c = float(x.reshape(-1)[0])
        ga, be = np.full(C, 2, np.float32), np.arange(C, dtype=np.float32) - 2
        X, GA, BE = DevArr(hip, x), DevArr(hip, ga), DevArr(hip, be)
        Y, M, R = DevArr(hip, shape=x.shape, fill=np.nan), DevArr(hip, shape=(N * G,), fill=np.nan), DevArr(hip, shape=(N * G,), fill=np.nan)
        hip.group_norm_fwd(0, hip.group_norm_desc(N, C, HW, G, last, 0, 0.0, eps), X.ptr, GA.ptr, BE.ptr, Y.ptr, M.ptr, R.ptr)
        m, r = M.get(), R.get()
        dm = (nb.H + 8 * nb.J) * nb.U * abs(c)
        rel = ((nb.H + 8 * nb.J) / 2 + 8) * nb.U
        assert (np.abs(m - c) <= dm).all()
        e32 = float(np.float32(eps))
        assert (r <= (1 + rel) / np.sqrt(e32)).all() and (r >= (1 - rel) / np.sqrt(e32 + (2 * dm) ** 2)).all()
        ry, ey = nb.Pass(x, ga, be, m, r, N, C, HW, G, last, 'none', 1.0).forward()
        y = Y.get()
        assert (np.abs(y - ry) <= ey).all()
        want = be if last else be[:, None]
        assert (np.abs(y - want) <= 2 * dm / np.sqrt(e32) * (1 + rel) + ey).all()
