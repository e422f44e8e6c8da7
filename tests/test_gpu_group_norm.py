"""lnn_group_norm_fwd_f32 / _bwd_f32 through the C ABI against the 64-bit formulas.

Tolerances, from the arithmetic (u = 2^-24, h additions in the longest chain of any sum: no variant adds more than
D / 64 + 64 terms of a row one after the other, nor N + HW / 64 + 64 for a channel):
  forward   |dmean| <= h u max|x|, so |d xh| <= (h + 4) u max|x| rstd + h u |xh|;  |f'| <= 1.1 and 8 more roundings:
            |dy| <= 1.1 (h + 8) u (|gamma| (max|x| rstd + |xh|) + |beta|)
  backward  every term of dx carries |gamma dy| times at most (1 + |xh|)^2 and, through xh and f'' <= 0.5, the error of xh
            above:  |d dx| <= (h + 32) u rstd max|gamma dy| (1 + max|xh|)^2 (1 + max|gamma|) (1 + max|x| rstd)
            dgamma, dbeta: the same without rstd gamma, summed over the channel's terms
Where the activation's slope jumps (leaky ReLU at 0) an element whose p lies within the error of p of 0 may take either
slope; such elements are left out of dx and their whole contribution is allowed in the sums."""
import itertools

import numpy as np
import pytest

from oracle.group_norm import act, group_norm_bwd, group_norm_fwd
from oracle.keep8 import keep8_encode, keep8_pack, keep8_values
from tests.gpu_util import DevArr, say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTS = {'none': 0, 'leaky_relu': 1, 'silu': 2}


def bytes_dev(api, data):
    """Bytes (uint8 array) on the device."""
    data = np.concatenate([data, np.zeros(-data.size % 4, np.uint8)])
    return DevArr(api, data.view(np.float32))


def make(seed, N, C, HW, last, offset=0.5, scale=1.0):
    rs = np.random.RandomState(seed)
    shape, per_c = ((N, HW, C), (1, 1, C)) if last else ((N, C, HW), (1, C, 1))
    x = (rs.normal(0, scale, shape) * np.exp(rs.normal(0, 0.3, per_c)) + offset * rs.normal(0, 1, per_c)).astype(np.float32)
    dy = rs.normal(0, 1, shape).astype(np.float32)
    return x, dy, rs.normal(1, 0.3, C).astype(np.float32), rs.normal(0, 0.3, C).astype(np.float32)


def check(api, seed, N, C, HW, groups, last, name, slope=0.1, eps=1e-5, kept=False, affine=True, prefill=None, x=None, offset=0.5):
    say(f'group_norm N={N} C={C} HW={HW} groups={groups} last={last} act={name} kept={kept} affine={affine} prefill={prefill}')
    made, dy, gamma, beta = make(seed, N, C, HW, last, offset)
    x = made if x is None else x
    if not affine:
        gamma = beta = None
    D, rows = C // groups * HW, N * groups
    desc = api.group_norm_desc(N, C, HW, groups, last, ACTS[name], slope, eps)
    X, dY = DevArr(api, x), DevArr(api, dy)
    GA, BE = (DevArr(api, gamma), DevArr(api, beta)) if affine else (None, None)
    ga, be = (GA.ptr, BE.ptr) if affine else (None, None)
    Y, M, R = DevArr(api, shape=x.shape, fill=np.nan), DevArr(api, shape=(rows,), fill=np.nan), DevArr(api, shape=(rows,), fill=np.nan)
    X8 = DevArr(api, shape=((api.bytes8(x.size) + 3) // 4,), fill=np.nan) if kept else None
    api.group_norm_fwd(0, desc, X.ptr, ga, be, Y.ptr, M.ptr, R.ptr, X8.ptr if kept else None)
    ry, rm, rr = group_norm_fwd(x, gamma, beta, N, C, HW, groups, last, name, slope, eps)
    h = D / 64 + 64
    gm, bm = (np.abs(gamma).max(), np.abs(beta).max()) if affine else (1.0, 0.0)
    amax = float(np.abs(x).max())
    rs_max = rr.max()
    y, mean, rstd = Y.get(), M.get(), R.get()
    assert np.abs(mean - rm.reshape(-1)).max() <= h * U * amax
    # relative error of var + eps: that of the squares' sum plus the mean's error, which enters squared
    assert (np.abs(rstd / rr.reshape(-1) - 1) <= (h + 8) * U + (h * U * amax * rs_max) ** 2).all()
    xh_max = np.sqrt(D)      # |xh| of any row
    xh_max = min(xh_max, (np.abs(x).max() + np.abs(rm).max()) * rs_max)
    xh_err = (h + 4) * U * amax * rs_max + h * U * xh_max
    assert np.abs(y - ry).max() <= 1.1 * (h + 8) * U * (gm * (amax * rs_max + xh_max) + bm)
    xs = x
    if kept:
        raw = X8.get().view(np.uint8)[:api.bytes8(x.size)]
        assert np.array_equal(raw, keep8_pack(*keep8_encode(x)))
        xs = keep8_values(x)
    outs = [DevArr(api, shape=s, fill=np.nan if prefill is None else prefill) for s in (x.shape, (C,), (C,))]
    b = 0 if prefill is None else 1
    api.group_norm_bwd(0, desc, None if kept else X.ptr, X8.ptr if kept else None, ga, be, M.ptr, R.ptr, dY.ptr,
                       outs[0].ptr, outs[1].ptr, outs[2].ptr, b, b, b)
    base = 0.0 if prefill is None else prefill
    ref = group_norm_bwd(xs, dy, gamma, beta, mean.reshape(N, groups), rstd.reshape(N, groups), N, C, HW, groups, last, name, slope)
    dmax = float(np.abs(dy).max())
    xh_max = np.abs(xs).max() * rs_max + np.abs(rm).max() * rs_max
    c = (1 + xh_max) ** 2 * (1 + gm) * (1 + amax * rs_max)
    tols = [(h + 32) * U * rs_max * gm * dmax * c, (N + HW / 64 + 96) * U * dmax * c * N * HW, (N + HW / 64 + 96) * U * dmax * c * N * HW]
    near = np.zeros(x.shape, bool)
    if name == 'leaky_relu':
        g64 = np.ones(C) if gamma is None else gamma
        shape = (1, 1, C) if last else (1, C, 1)

        def per_row(v):     # (N, groups) -> per element
            v = np.repeat(v.reshape(N, groups), C // groups, 1)
            return v[:, None, :] if last else v[:, :, None]
        p = (xs.astype(np.float64) - per_row(mean)) * per_row(rstd) * g64.reshape(shape) + (0 if beta is None else beta.reshape(shape))
        near = np.abs(p) <= 16 * U * (gm * (amax * rs_max + xh_max) + bm)
        tols = [tols[0] + near.sum() * gm * dmax * rs_max * (1 + xh_max ** 2) / D] + [t + near.sum() * dmax * (1 + xh_max) for t in tols[1:]]
    for what, o, r, tol in zip(('dx', 'dgamma', 'dbeta'), outs, ref, tols):
        err = np.abs(o.get() - base - r)
        if what == 'dx':
            err[near] = 0
        # an accumulated result is rounded once more, at the size of what was there
        assert err.max() <= tol + abs(base) * U * 4 + np.abs(r).max() * U, (what, err.max(), tol)
    # each gradient alone gives the same bits
    if prefill is None:
        alone = [DevArr(api, shape=s, fill=np.nan) for s in (x.shape, (C,), (C,))]
        for k in range(3):
            p = [a.ptr if i == k else None for i, a in enumerate(alone)]
            api.group_norm_bwd(0, desc, None if kept else X.ptr, X8.ptr if kept else None, ga, be, M.ptr, R.ptr, dY.ptr, *p)
        for a, o in zip(alone, outs):
            assert np.array_equal(a.get(), o.get())
    return y


SHAPES = [  # N, C, HW, groups
    (1, 1, 3, 1), (1, 8, 1, 1), (1, 64, 196, 8), (2, 6, 35, 3), (3, 60, 37 * 41, 12), (2, 32, 64, 32), (1, 4, 63, 2), (5, 12, 9, 4),
    (2, 128, 56 * 56, 32), (1, 3, 1000, 1), (4, 96, 49, 8), (2, 320, 256, 32), (1, 16, 70 * 71, 1), (2, 40, 33, 5), (7, 24, 1, 3),
    (300, 96, 1, 4), (33, 512, 1, 32), (64, 1000, 1, 1), (9, 34, 2, 17), (2, 1028, 5, 4), (1, 2, 65536, 2), (1, 64, 16384, 2),
    (600, 8, 4, 2), (5, 2048, 1, 1), (3, 5000, 1, 1), (2, 20000, 1, 2), (3, 6, 90000, 3), (2, 8000, 3, 1), (1, 33, 70000, 1), (1, 2080, 40, 5),
    (1, 1, 1, 1), (1, 1, 2, 1), (1, 3, 1, 1), (50, 3, 1, 1), (50, 3, 1, 3), (9, 2, 1, 1), (40, 5, 1, 5), (2, 3, 9001, 1), (150, 8, 3001, 2),
    (260, 26, 1000, 1), (270, 26, 999, 1), (3, 7, 1, 1), (70, 1, 19, 1)]


@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('last', [False, True])
def test_group_norm(hip, shape, last):
    for name, kept in itertools.product(ACTS, [False, True]):
        check(hip, 1, *shape, last, name, kept=kept)


@pytest.mark.parametrize('last', [False, True])
def test_group_norm_accumulates_and_has_optional_parameters(hip, last):
    for shape in [(2, 6, 35, 3), (3, 64, 64, 8), (40, 64, 1, 8), (1, 8, 5000, 2)]:
        for kept in (False, True):
            check(hip, 2, *shape, last, 'silu', kept=kept, prefill=0.5)
        check(hip, 3, *shape, last, 'leaky_relu', slope=0.0, affine=False)
        check(hip, 4, *shape, last, 'none', affine=False, kept=True)
        check(hip, 5, *shape, last, 'leaky_relu', slope=-0.5)


@pytest.mark.parametrize('last', [False, True])
def test_group_norm_far_from_zero(hip, last):
    """Values around 1000 with a spread of 1: a variance taken as a difference of squares would have no digits left."""
    for shape in [(2, 8, 300, 2), (1, 64, 4096, 2), (200, 64, 1, 2), (1, 8, 70000, 2)]:
        N, C, HW, G = shape
        x = (make(6, N, C, HW, last, 0.0)[0] + 1000).astype(np.float32)
        check(hip, 6, *shape, last, 'none', x=x)


@pytest.mark.parametrize('last', [False, True])
def test_group_norm_constant_rows(hip, last):
    """No variance: xh is 0 and y is act(beta)."""
    for N, C, HW, G in [(2, 6, 10, 3), (1, 8, 9000, 2), (5, 16, 1, 4), (3, 4, 1, 4)]:
        say(f'group_norm constant {N} {C} {HW} {G} last={last}')
        x = np.full((N, C, HW), 3.25, np.float32)
        be = np.arange(C, dtype=np.float32) - 2
        X, GA, BE = DevArr(hip, x), DevArr(hip, np.full(C, 2, np.float32)), DevArr(hip, be)
        Y, M, R = DevArr(hip, shape=x.shape), DevArr(hip, shape=(N * G,)), DevArr(hip, shape=(N * G,))
        hip.group_norm_fwd(0, hip.group_norm_desc(N, C, HW, G, last, 0, 0.0, 1e-5), X.ptr, GA.ptr, BE.ptr, Y.ptr, M.ptr, R.ptr)
        want = np.broadcast_to(be if last else be[:, None], (N, HW, C) if last else (N, C, HW))
        assert np.array_equal(Y.get().reshape(want.shape), want)
        assert np.array_equal(M.get(), np.full(N * G, 3.25, np.float32))


@pytest.mark.parametrize('last', [False, True])
def test_group_norm_nonfinite_stays_in_its_row(hip, last):
    N, C, HW, G = 3, 64, 64, 4
    for bad, kept in itertools.product((np.nan, np.inf, -np.inf), (False, True)):
        say(f'group_norm nonfinite {bad} last={last} kept={kept}')
        x, dy, ga, be = make(7, N, C, HW, last)
        at = (1, 5, 20) if last else (1, 20, 5)       # image 1, channel 20: group 1
        x[at] = bad
        X, dY, GA, BE = (DevArr(hip, v) for v in (x, dy, ga, be))
        Y, M, R = DevArr(hip, shape=x.shape), DevArr(hip, shape=(N * G,)), DevArr(hip, shape=(N * G,))
        X8 = DevArr(hip, shape=((hip.bytes8(x.size) + 3) // 4,)) if kept else None
        dX = DevArr(hip, shape=x.shape)
        d = hip.group_norm_desc(N, C, HW, G, last, 2, 0.0, 1e-5)
        hip.group_norm_fwd(0, d, X.ptr, GA.ptr, BE.ptr, Y.ptr, M.ptr, R.ptr, X8.ptr if kept else None)
        hip.group_norm_bwd(0, d, None if kept else X.ptr, X8.ptr if kept else None, GA.ptr, BE.ptr, M.ptr, R.ptr, dY.ptr, dX.ptr,
                           None, None)
        for t in (Y.get(), dX.get()):
            t = (t.reshape(N, HW, G, C // G).transpose(0, 2, 1, 3) if last else t.reshape(N, G, C // G, HW)).reshape(N * G, -1)
            rows = np.isfinite(t).all(1)
            assert np.isnan(t[5]).any() and not rows[5]
            # a kept block that straddles rows would spread further; channels first, rows are whole blocks here
            assert last and kept or rows.sum() == N * G - 1


def test_group_norm_on_unaligned_pointers(hip):
    """Tensors at 4-byte alignment only."""
    for last, kept in itertools.product((False, True), (False, True)):
        for N, C, HW, G in [(2, 64, 64, 8), (2, 8, 5000, 2), (40, 128, 1, 4)]:
            say(f'group_norm unaligned {N} {C} {HW} {G} last={last} kept={kept}')
            x, dy, ga, be = make(8, N, C, HW, last)
            d = hip.group_norm_desc(N, C, HW, G, last, 2, 0.0, 1e-5)
            got = []
            for off in (0, 1):
                def up(a):
                    return DevArr(hip, np.concatenate([np.zeros(off, np.float32), a.reshape(-1)]))

                def room(n):
                    return DevArr(hip, shape=(n + off,), fill=7.0)
                o = 4 * off
                ins = [up(v) for v in (x, dy, ga, be)]
                Y, M, R, dX, dG, dB = (room(n) for n in (x.size, N * G, N * G, x.size, C, C))
                X8 = DevArr(hip, shape=((hip.bytes8(x.size) + 3) // 4 + 1,), fill=7.0) if kept else None
                x8 = X8.ptr + off if kept else None      # the copy may start at any byte
                hip.group_norm_fwd(0, d, ins[0].ptr + o, ins[2].ptr + o, ins[3].ptr + o, Y.ptr + o, M.ptr + o, R.ptr + o, x8)
                hip.group_norm_bwd(0, d, None if kept else ins[0].ptr + o, x8, ins[2].ptr + o, ins[3].ptr + o, M.ptr + o, R.ptr + o,
                                   ins[1].ptr + o, dX.ptr + o, dG.ptr + o, dB.ptr + o)
                full = [t.get() for t in (Y, M, R, dX, dG, dB)]
                assert all((t[:off] == 7.0).all() for t in full)      # nothing in front of the outputs was touched
                got.append([t[off:] for t in full])
            for a, b in zip(*got):
                # another alignment may take another variant, whose sums are ordered differently: both within the bounds of
                # the comparison above, so twice that of each other; here plainly a few roundings of the largest value
                assert np.abs(a - b).max() <= 64 * U * max(1.0, float(np.abs(a).max()))


def test_group_norm_repeats_bit_for_bit(hip):
    for shape, last in (((4, 64, 900, 8), False), ((4, 64, 900, 8), True), ((500, 64, 1, 8), True), ((1, 8, 100000, 1), True)):
        N, C, HW, G = shape
        say(f'group_norm repeat {shape} last={last}')
        x, dy, ga, be = make(9, N, C, HW, last)
        X, dY, GA, BE = (DevArr(hip, v) for v in (x, dy, ga, be))
        d = hip.group_norm_desc(N, C, HW, G, last, 2, 0.0, 1e-5)
        runs = []
        for _ in range(3):
            o = [DevArr(hip, shape=s, fill=np.nan) for s in (x.shape, (N * G,), (N * G,), x.shape, (C,), (C,))]
            hip.group_norm_fwd(0, d, X.ptr, GA.ptr, BE.ptr, o[0].ptr, o[1].ptr, o[2].ptr)
            hip.group_norm_bwd(0, d, X.ptr, None, GA.ptr, BE.ptr, o[1].ptr, o[2].ptr, dY.ptr, o[3].ptr, o[4].ptr, o[5].ptr)
            runs.append([t.get() for t in o])
        for r in runs[1:]:
            assert all(np.array_equal(a, b) for a, b in zip(runs[0], r))
