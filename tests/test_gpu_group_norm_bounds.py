"""lnn_group_norm_fwd_f32 / _bwd_f32 against the 64-bit formulas, every element of every output within a bound from its own
terms (tests/norm_bounds.py).  Each comparison first shows that its bounds would not let zeros pass."""
import numpy as np
import pytest

from oracle.keep8 import keep8_values
from tests import norm_bounds as nb
from tests.gpu_util import DevArr, say

pytestmark = pytest.mark.gpu
ACTS = {'none': 0, 'leaky_relu': 1, 'silu': 2}


def check(api, seed, N, C, HW, G, last, act, kept=False, slope=0.1, eps=1e-5, offset=None, add=None, lean=0.0):
    """offset: added to every x (None: 0.5 times a normal value of each channel).  add: accumulate onto this value.
    lean: how far dy leans to 1 and to x, so that sums over very many elements of few channels do not cancel."""
    say(f'bounds N={N} C={C} HW={HW} groups={G} last={last} act={act} kept={kept} offset={offset} add={add} lean={lean}')
    rs = np.random.RandomState(seed)
    shape, per_c = ((N, HW, C), (1, 1, C)) if last else ((N, C, HW), (1, C, 1))
    x = (rs.normal(0, 1, shape) + (0.5 * rs.normal(0, 1, per_c) if offset is None else offset)).astype(np.float32)
    dy = (rs.normal(0, 1, shape) + lean * (1 + x)).astype(np.float32)
    ga, be = rs.normal(1, 0.3, C).astype(np.float32), rs.normal(0, 0.3, C).astype(np.float32)
    d = api.group_norm_desc(N, C, HW, G, last, ACTS[act], slope, eps)
    X, dY, GA, BE = (DevArr(api, v) for v in (x, dy, ga, be))
    Y, M, R = DevArr(api, shape=shape, fill=np.nan), DevArr(api, shape=(N * G,), fill=np.nan), DevArr(api, shape=(N * G,), fill=np.nan)
    X8 = DevArr(api, shape=((api.bytes8(x.size) + 3) // 4,), fill=np.nan) if kept else None
    api.group_norm_fwd(0, d, X.ptr, GA.ptr, BE.ptr, Y.ptr, M.ptr, R.ptr, X8.ptr if kept else None)
    outs = [DevArr(api, shape=s, fill=np.nan if add is None else add) for s in (shape, (C,), (C,))]
    b = int(add is not None)
    api.group_norm_bwd(0, d, None if kept else X.ptr, X8.ptr if kept else None, GA.ptr, BE.ptr, M.ptr, R.ptr, dY.ptr,
                       *(o.ptr for o in outs), b, b, b)
    m, r = M.get(), R.get()
    mean, rstd, e_mean, e_rstd = nb.statistics(x, N, C, HW, G, last, eps)
    assert (np.abs(m - mean) <= e_mean).all() and (np.abs(r - rstd) <= e_rstd).all()
    s32 = float(np.float32(slope))
    ry, ey = nb.Pass(x, ga, be, m, r, N, C, HW, G, last, act, s32).forward()
    refs, bounds = nb.Pass(keep8_values(x) if kept else x, ga, be, m, r, N, C, HW, G, last, act, s32).backward(dy)
    if C // G * HW >= 8:      # a row of fewer elements can lose all of its gradient to cancellation
        assert nb.telling([ry], [ey])[0] and all(nb.telling(refs, bounds))
    assert (np.abs(Y.get() - ry) <= ey).all(), ('y', np.abs(Y.get() - ry).max())
    for what, o, ref, e in zip(('dx', 'dgamma', 'dbeta'), outs, refs, bounds):
        got = o.get()
        if add is not None:   # one more rounding, of the accumulated value
            ref = ref + add
            e = e + nb.U * np.abs(ref)
        off = np.abs(got - ref)
        assert (off <= e).all(), (what, off.max(), float(e.reshape(-1)[off.argmax()]))


SHAPES = [  # N, C, HW, groups: rows of channels; rows in registers; small channels last; split, with one and with two stages of channel sums
    (33, 512, 1, 32), (300, 96, 1, 4), (64, 1000, 1, 1), (5, 2048, 1, 1), (2, 20000, 1, 2), (9, 34, 2, 2),
    (2, 128, 56 * 56, 32), (3, 60, 37 * 41, 12), (2, 320, 256, 32), (1, 64, 16384, 2), (600, 8, 4, 2), (2, 1028, 5, 4),
    (3, 6, 90000, 3), (2, 8000, 3, 1), (1, 33, 70000, 1), (1, 2080, 40, 5), (40, 256, 196, 8), (700, 96, 50, 4), (260, 26, 1000, 1)]


@pytest.mark.parametrize('last', [False, True])
@pytest.mark.parametrize('shape', SHAPES)
def test_every_output_within_its_bound(hip, shape, last):
    for k, act in enumerate(ACTS):
        check(hip, 20 + k, *shape, last, act, kept=k % 2 == 1)
    check(hip, 23, *shape, last, 'silu', kept=True)
    check(hip, 24, *shape, last, 'silu', add=0.25)


@pytest.mark.parametrize('last', [False, True])
def test_far_from_zero(hip, last):
    for shape in [(2, 8, 300, 2), (1, 64, 4096, 2), (200, 64, 1, 2), (1, 8, 70000, 2)]:
        check(hip, 25, *shape, last, 'none', offset=1000.0)
        check(hip, 26, *shape, last, 'silu', offset=-300.0)
