"""The 64-bit restatements of group norm and of the 8-bit activation format, each pinned by something that does not use
its formula: torch's group norm and numerical differences; the format's error bound and properties."""
import numpy as np
import pytest

from oracle.group_norm import group_norm_bwd, group_norm_fwd
from oracle.keep8 import keep8_decode, keep8_encode, keep8_values


@pytest.mark.parametrize('last', [False, True])
@pytest.mark.parametrize('name', ['none', 'leaky_relu', 'silu'])
def test_group_norm_against_torch(name, last):
    import torch
    rs = np.random.RandomState(3)
    N, C, HW, G = 2, 6, 7, 3
    x, dy = rs.normal(1, 2, (N, C, HW)), rs.normal(0, 1, (N, C, HW))
    ga, be = rs.normal(1, 0.3, C), rs.normal(0, 0.3, C)
    tx, tg, tb = (torch.tensor(v, requires_grad=True) for v in (x, ga, be))
    p = torch.nn.functional.group_norm(tx, G, tg, tb, 1e-3)
    y = dict(none=lambda v: v, leaky_relu=lambda v: torch.nn.functional.leaky_relu(v, 0.2), silu=torch.nn.functional.silu)[name](p)
    y.backward(torch.tensor(dy))

    def lay(t):
        return np.ascontiguousarray(t.transpose(0, 2, 1)) if last else t
    ry, mean, rstd = group_norm_fwd(lay(x), ga, be, N, C, HW, G, last, name, 0.2, 1e-3)
    dx, dg, db = group_norm_bwd(lay(x), lay(dy), ga, be, mean, rstd, N, C, HW, G, last, name, 0.2)
    for got, ref in ((ry, lay(y.detach().numpy())), (dx, lay(tx.grad.numpy())), (dg, tg.grad.numpy()), (db, tb.grad.numpy())):
        assert np.abs(got - ref).max() <= 1e-12


def test_group_norm_gradient_by_differences():
    rs = np.random.RandomState(4)
    N, C, HW, G = 1, 4, 5, 2
    x, dy, ga, be = rs.normal(0, 1, (N, C, HW)), rs.normal(0, 1, (N, C, HW)), rs.normal(1, 0.2, C), rs.normal(0, 0.2, C)

    def loss(x, ga, be):
        return float((group_norm_fwd(x, ga, be, N, C, HW, G, False, 'silu', 0.0, 1e-3)[0] * dy).sum())
    _, mean, rstd = group_norm_fwd(x, ga, be, N, C, HW, G, False, 'silu', 0.0, 1e-3)
    grads = group_norm_bwd(x, dy, ga, be, mean, rstd, N, C, HW, G, False, 'silu', 0.0)
    h = 1e-6
    for k, (v, grad) in enumerate(zip((x, ga, be), grads)):
        for i in range(v.size):
            a, b = [t.copy() for t in (x, ga, be)], [t.copy() for t in (x, ga, be)]
            a[k].reshape(-1)[i] += h
            b[k].reshape(-1)[i] -= h
            # central differences: h^2 f'''/6 + rounding of the loss / h, both far below 1e-7 here
            assert abs((loss(*a) - loss(*b)) / (2 * h) - grad.reshape(-1)[i]) <= 1e-7


def test_keep8_error_and_range():
    rs = np.random.RandomState(5)
    x = (rs.normal(0, 1, 32 * 4000) * np.repeat(np.exp2(rs.uniform(-120, 120, 4000)), 32)).astype(np.float32)
    codes, byte = keep8_encode(x)
    v = keep8_decode(codes, byte, x.size).astype(np.float64)
    step = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32)
    assert (np.abs(v - x) <= step / 2).all()
    top = np.abs(codes.astype(int)).max(1)
    assert top.min() >= 64 and top.max() <= 127      # no block wastes a bit
    assert np.array_equal(keep8_values(v), v.astype(np.float32))   # what was kept once is kept exactly
    assert np.array_equal((v.astype(np.float32).view(np.uint32) & 0xffff), np.zeros(v.size, np.uint32))  # bf16 numbers


def test_keep8_edges():
    def one(*vals):
        x = np.zeros(32, np.float32)
        x[:len(vals)] = vals
        c, b = keep8_encode(x)
        return c[0], int(b[0]), keep8_decode(c, b, 32)
    assert one()[1] == 0 and not one()[2].any()
    c, b, v = one(127.5)            # would round to 128 with step 1
    assert b == 128 and c[0] == 64 and v[0] == 128.0
    c, b, v = one(np.nextafter(np.float32(127.5), np.float32(0)))
    assert b == 127 and c[0] == 127
    c, b, v = one(127, 2.5, 3.5, -2.5)   # ties go to the even code
    assert list(c[1:4]) == [2, 4, -2]
    fmax = np.finfo(np.float32).max
    c, b, v = one(fmax, -fmax)      # saturates instead of overflowing
    assert b == 248 and list(c[:2]) == [127, -127] and np.isfinite(v).all()
    c, b, v = one(np.float32(1e-45), np.float32(2.0 ** -126))
    assert b == 1 and list(c[:2]) == [0, 1]
    for bad in (np.nan, np.inf, -np.inf):
        c, b, v = one(1.0, bad)
        assert b == 255 and not c.any() and np.isnan(v).all()
