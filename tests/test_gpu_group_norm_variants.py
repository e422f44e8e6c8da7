"""Group norm on a shape of every kernel variant, with its row as long as the variant holds and ragged, against the per-element
bounds of tests/norm_bounds.py."""
import numpy as np
import pytest

from litenn_amd.core.hip import api
from tests.test_gpu_group_norm_bounds import check
from tests.test_group_norm_plan import GATHER, RES_BWD, RES_FWD, ROWS

pytestmark = pytest.mark.gpu


def path(hip, shape, last, backward, kept=False):
    return hip.group_norm_path(hip.group_norm_desc(*shape, last), backward, kept, hip.device_info(0)['compute_units'])


@pytest.mark.parametrize('T,V', GATHER)
def test_gathered_rows(hip, T, V):
    """Channels last: for wide and narrow groups the fewest and the most pixels that the variant serves."""
    ran = 0
    for cg, groups in ((1, 5), (20, 3), (48, 2), (100, 1), (160, 2), (256, 1)):
        served = [hw for hw in range(2, 1024 // cg * 16 + 1) if path(hip, (2, cg * groups, hw, groups), True, False) == (api.NORM_PATH_GATHERED_ROW, T, V)]
        for hw in sorted({served[0], served[-1]}) if served else ():
            shape = (2, cg * groups, hw, groups)
            assert path(hip, shape, True, True) == (api.NORM_PATH_GATHERED_ROW, T, V)
            check(hip, 30, *shape, True, 'silu')
            check(hip, 31, *shape, True, 'leaky_relu', kept=True, add=0.5)
            ran += 1
    assert ran


@pytest.mark.parametrize('shape', [(4, 640, 14 * 14, 32), (2, 1280, 10 * 10, 32), (8, 384, 9 * 9, 8), (2, 100, 36, 1), (1, 160, 20, 1),
                                   (3, 52, 70, 1), (1, 3, 1361, 1)])
def test_between_the_variants(hip, shape):
    for kept in (False, True):
        check(hip, 32, *shape, True, 'silu', kept=kept)
    check(hip, 38, *shape, True, 'none', offset=1000.0)


@pytest.mark.parametrize('shape', [(4, 640, 14, 14), (2, 1280, 10, 10), (8, 384, 9, 9)])
def test_between_the_variants_through_tensors(nn_hip, shape):
    """The calls as a program makes them, channels last against the same norm channels first."""
    nn = nn_hip
    N, C = shape[:2]
    rs = np.random.RandomState(33)
    x, dy = rs.normal(0, 1, shape).astype(np.float32), rs.normal(0, 1, shape).astype(np.float32)
    got = []
    for last in (False, True):
        def lay(v):
            return np.ascontiguousarray(np.moveaxis(v, 1, -1)) if last else v
        x_t = nn.Tensor_from_value(lay(x))
        y_t = nn.group_norm(x_t, 32, activation='silu', channels_last=last)
        nn.backward({y_t: lay(dy)}, grad_for_non_trainables=True)
        got.append([np.moveaxis(v, -1, 1) if last else v for v in (y_t.np(), x_t.get_grad().np())])
    for a, b in zip(*got):
        # each within 2^-16 of the definition at values of a few units: sums of at most 10^4 terms in short chains
        assert np.abs(a - b).max() <= 2.0 ** -15 * np.abs(a).max()


@pytest.mark.parametrize('L,V', ROWS)
def test_rows_of_channels(hip, L, V):
    served = [cg for cg in range(1, 8193) if path(hip, (2, cg, 1, 1), False, False) == (api.NORM_PATH_ROWS, L, V)]
    for cg in sorted({served[0], served[-1], max(served[0], served[-1] - 1)}):
        groups = 3 if cg < 2000 else 1
        for N in (1, 70):
            check(hip, 34, N, cg * groups, 1, groups, N == 1, 'silu')
        check(hip, 35, 9, cg * groups, 1, groups, False, 'none', kept=True)


@pytest.mark.parametrize('T,V', RES_FWD)
def test_rows_in_registers(hip, T, V):
    """Channels first: the longest row, forward and backward from fp32 or 8 bits, and one of ragged planes."""
    cus = hip.device_info(0)['compute_units']
    served = 0
    for N, HW in ((3, 4 * T * V), (cus + 1, 4 * T * V)):
        for kept in (False, True):
            f, b = (path(hip, (N, 1, HW, 1), False, k, kept) == (api.NORM_PATH_ROW_IN_REGISTERS, T, V) for k in (False, True))
            if not (f or b) or (served and N > 3):
                continue
            served += 1
            check(hip, 36, N, 1, HW, 1, False, 'silu', kept=kept, lean=0.5)
            if HW > 64:
                # three channels of ragged planes, the row in the same variant where it allows that
                check(hip, 37, N if N == 3 else 90, 3, HW // 3 - 1, 1, False, 'leaky_relu', kept=kept, lean=0.5)
    assert served
    # the backward pass has its variant from somewhere too
    if (T, V) in RES_BWD:
        assert any(path(hip, (n, 1, 4 * T * V, 1), False, True, k) == (api.NORM_PATH_ROW_IN_REGISTERS, T, V)
                   for n in (3, cus + 1) for k in (False, True))
