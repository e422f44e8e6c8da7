"""An infinity or NaN in the first block of an 8-bit copy: lanes without elements read that block, and nothing of it may
reach a result.  The rows and channels that the block belongs to become NaN, and no others."""
import itertools

import numpy as np
import pytest

from oracle.keep8 import keep8_values
from tests import norm_bounds as nb
from tests.gpu_util import DevArr, say
from tests.test_gpu_keep8 import wgrad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('bad', [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize('shape', [  # batch, rows, K, M: rows not whole steps, K whole groups of four and not, one and several tiles
    (2, 70, 96, 40), (1, 1, 64, 8), (3, 33, 32, 130), (1, 1000, 300, 33), (2, 70, 35, 40), (1, 515, 260, 700), (3, 7, 4, 3)])
def test_weight_gradient(hip, shape, bad):
    batch, rows, K, M = shape
    say(f'wgrad8 bad first block {shape} {bad}')
    rs = np.random.RandomState(40)
    x, dy = rs.randint(-15, 16, (batch, rows, K)).astype(np.float32), rs.randint(-8, 9, (batch, rows, M)).astype(np.float32)
    x[0, 0, 0] = bad
    v = keep8_values(x)
    assert np.isnan(v.reshape(-1)[:32]).all() and np.isfinite(v.reshape(-1)[32:]).all()
    with np.errstate(invalid='ignore'):
        ref = np.matmul(v.transpose(0, 2, 1).astype(np.float64), dy.astype(np.float64))
    assert np.isfinite(ref).any()
    # whole numbers below 2^24: exact in any order
    assert np.array_equal(wgrad(hip, x, dy), ref, equal_nan=True)
    assert np.array_equal(wgrad(hip, x, dy, prefill=2.0), ref + 2, equal_nan=True)


SHAPES = [  # N, C, HW, groups, last: sums over pixels that are not whole tiles and over several images
    (3, 64, 20001, 4, True), (2, 96, 16383, 3, True), (40, 320, 333, 32, True), (2, 66, 9001, 3, True), (3, 1028, 400, 4, True),
    (3, 8, 50001, 2, False), (2, 4, 66000, 2, False), (5, 64, 100, 4, False), (3, 64, 37, 4, True), (70, 64, 1, 4, False), (33, 130, 1, 2, True)]


@pytest.mark.parametrize('bad', [np.nan, np.inf])
@pytest.mark.parametrize('shape', SHAPES)
def test_group_norm(hip, shape, bad):
    """The bad block lies in image 0, group 0 or (channels last, in small groups) a few groups behind it."""
    N, C, HW, G, last = shape
    say(f'group_norm bad first block {shape} {bad}')
    rs = np.random.RandomState(41)
    tshape = (N, HW, C) if last else (N, C, HW)
    x, dy = rs.normal(0, 1, tshape).astype(np.float32), (rs.normal(0, 1, tshape) + 0.5).astype(np.float32)
    ga, be = rs.normal(1, 0.3, C).astype(np.float32), rs.normal(0, 0.3, C).astype(np.float32)
    # the statistics that a forward pass left before the value went bad: what is tested is the backward pass
    mean, rstd, _, _ = nb.statistics(x, N, C, HW, G, last, 1e-5)
    m32, r32 = mean.astype(np.float32), rstd.astype(np.float32)
    x.reshape(-1)[0] = bad
    d = hip.group_norm_desc(N, C, HW, G, last, 2, 0.0, 1e-5)
    dY, GA, BE, M, R, X = (DevArr(hip, v) for v in (dy, ga, be, m32, r32, x))
    X8 = DevArr(hip, shape=((hip.bytes8(x.size) + 3) // 4,), fill=np.nan)
    hip.encode8(0, x.size, X.ptr, X8.ptr)
    outs = [DevArr(hip, shape=s, fill=7.0) for s in (tshape, (C,), (C,))]
    hip.group_norm_bwd(0, d, None, X8.ptr, GA.ptr, BE.ptr, M.ptr, R.ptr, dY.ptr, *(o.ptr for o in outs))
    with np.errstate(invalid='ignore'):
        refs, bounds = nb.Pass(keep8_values(x), ga, be, m32, r32, N, C, HW, G, last, 'silu', 0.0).backward(dy)
    for what, o, ref, e in zip(('dx', 'dgamma', 'dbeta'), outs, refs, bounds):
        got, fine = o.get(), np.isfinite(ref)
        assert fine.any() and np.array_equal(np.isfinite(got), fine), (what, np.isfinite(got).sum(), fine.sum())
        assert (np.abs(got - ref)[fine] <= e[fine]).all(), what


def test_shapes_reach_every_path(hip):
    """The shapes above take each of the four paths, and the split kernels in both layouts with whole groups and without."""
    cus = hip.device_info(0)['compute_units']
    got = set()
    for N, C, HW, G, last in SHAPES:
        path = hip.group_norm_path(hip.group_norm_desc(N, C, HW, G, last), True, True, cus)[0]
        got.add((path, last if HW > 1 else None, (C if last else HW) % 4 == 0) if path == hip.NORM_PATH_SPLIT else path)
    want = {(hip.NORM_PATH_SPLIT, last, four) for last, four in itertools.product((False, True), repeat=2)}
    assert got >= want | {hip.NORM_PATH_ROWS, hip.NORM_PATH_ROW_IN_REGISTERS, hip.NORM_PATH_GATHERED_ROW}
