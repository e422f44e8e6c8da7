"""Which kernels serve a group norm (lnn_group_norm_path: host arithmetic, no device needed).  Every legal problem has a plan whose
kernel holds its row, and every variant that is built serves some problem."""
import numpy as np
import pytest

from litenn_amd.core.hip import api

CUS = 256
RES_BWD = ([(64, 1)] + [(256, v) for v in (1, 2, 3, 4)] + [(512, v) for v in (3, 4, 5, 6, 7, 8, 10, 13)] +
           [(1024, v) for v in (2, 3, 4, 5, 6, 7, 8)])
RES_FWD = RES_BWD + [(512, 16), (1024, 10), (1024, 13), (1024, 16)]
ROWS = [(4, 1), (16, 1), (32, 1), (64, 1), (64, 2), (64, 4), (256, 2), (256, 4), (256, 8)]
GATHER = [(256, 1), (256, 4), (256, 8), (256, 16), (1024, 4), (1024, 8), (1024, 16)]


def plan(N, C, HW, G, last, backward=False, kept=False, cus=CUS):
    path, T, V = api.group_norm_path(api.group_norm_desc(N, C, HW, G, last), backward, kept, cus)
    return path, (T, V)


def test_small_channels_last():
    """Every number of channels to a group and of pixels that a workgroup can hold."""
    seen = set()
    for cg in range(1, 257):
        most = 1024 // cg * 16
        for hw in range(2, most + 2):
            for backward in (False, True):
                path, (T, V) = plan(1, 2 * cg, hw, 2, True, backward)
                fits = hw <= max(most, 256 // cg * 16)
                assert path == (api.NORM_PATH_GATHERED_ROW if fits else api.NORM_PATH_SPLIT), (cg, hw)
                if fits:
                    assert (T, V) in GATHER and T // cg * V >= hw, (cg, hw, T, V)
                    seen.add((T, V))
    assert seen == set(GATHER)
    # a tensor of more than 2^20 elements, and wide groups, are split
    assert plan(2, 512, 1025, 32, True)[0] == api.NORM_PATH_SPLIT
    assert plan(1, 257, 4, 1, True)[0] == api.NORM_PATH_SPLIT


@pytest.mark.parametrize('shape', [(4, 640, 14 * 14, 32), (2, 1280, 10 * 10, 32), (8, 384, 9 * 9, 8), (2, 100, 36, 1), (1, 160, 20, 1),
                                   (3, 52, 70, 1), (1, 3, 1361, 1)])
def test_between_the_variants(shape):
    for backward in (False, True):
        path, (T, V) = plan(*shape, True, backward)
        assert path == api.NORM_PATH_GATHERED_ROW and T // (shape[1] // shape[3]) * V >= shape[2]


def test_rows_of_channels():
    seen = set()
    for cg in range(1, 8300):
        for backward in (False, True):
            path, (L, V) = plan(3, cg, 1, 1, bool(cg & 1), backward)
            if cg <= 8192:
                assert path == api.NORM_PATH_ROWS and (L, V) in ROWS and 4 * L * V >= cg
                seen.add((L, V))
            else:
                assert path == api.NORM_PATH_SPLIT
    assert seen == set(ROWS)


def test_channels_first():
    """Random and systematic rows: a plan in registers has room for every unit of the row."""
    rs = np.random.RandomState(1)
    seen = {False: set(), True: set()}
    cases = [(n, 1, hw) for n in (1, 300) for hw in range(2, 66000, 37)]
    cases += [(int(n), int(cg), int(hw)) for n, cg, hw in zip(rs.choice([1, 40, 300], 20000), np.exp(rs.uniform(0, 9, 20000)), np.exp(rs.uniform(0.7, 12, 20000)))]
    for N, cg, hw in cases:
        if hw < 2 or N * cg * hw >= 1 << 29:
            continue
        for backward in (False, True):
            for kept in (False, True):
                path, (T, V) = plan(N, cg, hw, 1, False, backward, kept)
                ul = 0 if hw <= 4 else 2 if hw <= 16 else 4 if hw <= 64 else 6
                units = cg * -(-hw // (4 << ul))
                if path == api.NORM_PATH_ROW_IN_REGISTERS:
                    assert (T, V) in (RES_BWD if backward else RES_FWD) and units << ul <= T * V and units <= 3500, (N, cg, hw, T, V)
                    seen[backward].add((T, V))
                else:
                    lanes = units << ul
                    # 1024 lanes hold eight groups of four each at least; forward, 16, or 13 where planes are not whole groups
                    assert path == api.NORM_PATH_SPLIT and (units > 3500 or lanes > 1024 * (8 if backward else 16 if hw % 4 == 0 else 13))
    assert seen[False] == set(RES_FWD) and seen[True] == set(RES_BWD)


def test_few_rows_get_more_lanes():
    assert plan(1, 1, 8192, 1, False)[1] == (1024, 2)
    assert plan(CUS + 1, 1, 8192, 1, False)[1] == (512, 4)
    assert plan(CUS + 1, 1, 8192, 1, False, cus=304)[1] == (1024, 2)


def test_refusals():
    for d in (api.group_norm_desc(1, 4, 4, 3), api.group_norm_desc(0, 4, 4, 2), api.group_norm_desc(1, 4, 4, 2, eps=0.0)):
        with pytest.raises(api.HipException) as e:
            api.group_norm_path(d, False, False, CUS)
        assert e.value.code == api.ERR_INVALID
    with pytest.raises(api.HipException):
        api.group_norm_path(api.group_norm_desc(1, 4, 4, 2), False, False, 0)
