"""tests/norm_bounds.py itself, on the CPU: its formulas are the oracle's, a 32-bit evaluation lies within its bounds, and
results with a mistake in them do not."""
import numpy as np
import pytest

from oracle.group_norm import group_norm_bwd, group_norm_fwd
from tests import norm_bounds as nb

CASES = [  # N, C, HW, groups, offset: a row in registers, one gathered, rows of channels, split (long rows, many images)
    (2, 16, 3136, 4, 0.5), (3, 60, 1517, 12, 0.5), (300, 96, 1, 4, 0.5), (2, 6, 30000, 3, 0.5), (2, 300, 49, 1, 0.5),
    (700, 32, 16, 4, 0.5), (4, 64, 300, 4, 1000.0), (9, 34, 2, 2, 0.5), (1, 2, 4, 1, 0.0)]


def in_32_bits(x, dy, ga, be, mean, rstd, N, C, HW, G, last, act, slope):
    """A plain evaluation in float32, sums by numpy (pairwise)."""
    f = np.float32

    def rows(a):
        return np.ascontiguousarray(nb.rows_of(a, N, C, HW, G, last).astype(f))
    m, r = (np.asarray(v, f).reshape(N, G, 1, 1) for v in (mean, rstd))
    ga, be = ga.astype(f).reshape(1, G, -1, 1), be.astype(f).reshape(1, G, -1, 1)
    xh = (rows(x) - m) * r
    p = xh * ga + be
    d = rows(dy)
    if act == 'silu':
        s = f(1) / (f(1) + np.exp(-p))
        y, dp = p * s, d * (s + p * s * (f(1) - s))
    elif act == 'leaky_relu':
        y, dp = np.where(p >= 0, p, f(slope) * p), np.where(p >= 0, d, f(slope) * d)
    else:
        y, dp = p, d
    g = dp * ga
    D = f(C // G * HW)
    s1, s2 = g.sum((2, 3), keepdims=True) / D, (g * xh).sum((2, 3), keepdims=True) / D
    dx = r * (g - s1 - xh * s2)
    return y, dx, xh, dp, s1, s2


def inputs(seed, N, C, HW, offset):
    rs = np.random.RandomState(seed)
    x = (rs.normal(0, 1, (N, C, HW)) + offset * (1 if offset > 100 else rs.normal(0, 1, (1, C, 1)))).astype(np.float32)
    return x, rs.normal(0, 1, (N, C, HW)).astype(np.float32), rs.normal(1, 0.3, C).astype(np.float32), rs.normal(0, 0.3, C).astype(np.float32)


@pytest.mark.parametrize('act', ['none', 'leaky_relu', 'silu'])
@pytest.mark.parametrize('case', CASES)
def test_bounds(case, act):
    N, C, HW, G, offset = case
    slope = float(np.float32(0.1))
    x, dy, ga, be = inputs(1, N, C, HW, offset)
    mean, rstd, e_mean, e_rstd = nb.statistics(x, N, C, HW, G, False, 1e-5)
    m32, r32 = mean.astype(np.float32), rstd.astype(np.float32)
    assert (np.abs(m32 - mean) <= e_mean).all() and (np.abs(r32 - rstd) <= e_rstd).all()
    ps = nb.Pass(x, ga, be, m32, r32, N, C, HW, G, False, act, slope)
    (ry, ey), (refs, bounds) = ps.forward(), ps.backward(dy)
    # the formulas are the oracle's
    oy, om, orr = group_norm_fwd(x, ga, be, N, C, HW, G, False, act, slope, 1e-5)
    assert np.allclose(om.reshape(-1), mean, rtol=1e-12) and np.allclose(orr.reshape(-1), rstd, rtol=1e-12)
    for a, b in zip(refs, group_norm_bwd(x, dy, ga, be, m32.reshape(N, G), r32.reshape(N, G), N, C, HW, G, False, act, slope)):
        assert np.abs(a - b).max() <= 1e-11 * max(1.0, np.abs(b).max())
    # 32 bits lie within
    y, dx, xh, dp, s1, s2 = in_32_bits(x, dy, ga, be, m32, r32, N, C, HW, G, False, act, slope)
    got = [dx.reshape(refs[0].shape), (dp * xh).sum((0, 3)).reshape(-1), dp.sum((0, 3)).reshape(-1)]
    assert (np.abs(y.reshape(ry.shape) - ry) <= ey).all()
    for v, r, e in zip(got, refs, bounds):
        assert (np.abs(v - r) <= e).all()
    if C // G * HW < 8:
        return
    # mistakes do not: zeros, gammas and betas exchanged, the last pixels or images left out, a sum left out
    assert all(nb.telling(refs, bounds)) and nb.telling([ry], [ey])[0]
    assert (np.abs(refs[1] - refs[2]) > bounds[1]).any()
    last = 1 if HW == 1 else HW // 8 or 1
    dp_short = dp.copy()
    if HW == 1:
        dp_short[-1] = 0
    else:
        dp_short[..., -last:] = 0
    for t, k in ((dp_short, 2), (dp_short * xh, 1)):
        assert (np.abs(t.sum((0, 3)).reshape(-1) - refs[k]) > bounds[k]).any()
    r = r32.reshape(N, G, 1, 1)
    g = dp * ga.reshape(1, G, -1, 1)
    for wrong in (r * (g - xh * s2), r * (g - s1), r * g):
        assert (np.abs(wrong.reshape(refs[0].shape) - refs[0]) > bounds[0]).any()
