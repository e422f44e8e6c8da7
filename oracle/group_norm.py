"""Group normalisation with an activation, forward and backward, in 64 bits from its formulas (no reference file: the
reference has no group norm)."""
import numpy as np


def _rows(t, N, C, HW, groups, last):
    """(N, groups, channels of a group, pixels) view of a tensor stored channels first or last."""
    t = np.asarray(t, np.float64).reshape((N, HW, C) if last else (N, C, HW))
    return (t.transpose(0, 2, 1) if last else t).reshape(N, groups, C // groups, HW)


def _back(t, N, C, HW, last):
    t = t.reshape(N, C, HW)
    return np.ascontiguousarray(t.transpose(0, 2, 1)) if last else t


def act(p, name, slope):
    """f(p), f'(p) of 'none', 'leaky_relu' and 'silu'."""
    if name == 'leaky_relu':
        return np.where(p >= 0, p, slope * p), np.where(p >= 0, 1.0, slope)
    if name == 'silu':
        with np.errstate(over='ignore'):
            s = 1 / (1 + np.exp(-p))
        return p * s, s * (1 + p * (1 - s))
    return p, np.ones_like(p)


def group_norm_fwd(x, gamma, beta, N, C, HW, groups, last, name, slope, eps):
    """y (as x is stored), mean (N, groups), rstd (N, groups)."""
    r = _rows(x, N, C, HW, groups, last)
    mean = r.mean((2, 3))
    rstd = 1 / np.sqrt(((r - mean[..., None, None]) ** 2).mean((2, 3)) + eps)
    ga = np.ones(C) if gamma is None else np.asarray(gamma, np.float64)
    be = np.zeros(C) if beta is None else np.asarray(beta, np.float64)
    p = (r - mean[..., None, None]) * rstd[..., None, None] * ga.reshape(1, groups, -1, 1) + be.reshape(1, groups, -1, 1)
    return _back(act(p, name, slope)[0], N, C, HW, last), mean, rstd


def group_norm_bwd(x, dy, gamma, beta, mean, rstd, N, C, HW, groups, last, name, slope):
    """dx (as x is stored), dgamma (C,), dbeta (C,) for the statistics of the forward pass."""
    r, d = _rows(x, N, C, HW, groups, last), _rows(dy, N, C, HW, groups, last)
    ga = (np.ones(C) if gamma is None else np.asarray(gamma, np.float64)).reshape(1, groups, -1, 1)
    be = (np.zeros(C) if beta is None else np.asarray(beta, np.float64)).reshape(1, groups, -1, 1)
    rs = np.asarray(rstd, np.float64)[..., None, None]
    xh = (r - np.asarray(mean, np.float64)[..., None, None]) * rs
    dp = d * act(xh * ga + be, name, slope)[1]
    g = dp * ga
    dx = rs * (g - g.mean((2, 3), keepdims=True) - xh * (g * xh).mean((2, 3), keepdims=True))
    return _back(dx, N, C, HW, last), (dp * xh).sum((0, 3)).reshape(C), dp.sum((0, 3)).reshape(C)
