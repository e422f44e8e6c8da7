"""Group norm in 64 bits with a bound for every element of every output of a 32-bit evaluation, each from its own terms.

u = 2^-24 is the most that one rounding can be off, relative to its result; a one-instruction reciprocal or power of two 2u.
H additions follow each other at most in any sum: 64 within a lane, 16 across lanes and wavefronts, 128 units of a plane, 160
for the rows of a channel's sums (64 + 64 + two joins) - 368 in all, H = 400.  J statistics are joined one after the other at
most (4 groups of pixels, 8 rows of lanes, 128 chunks, 22 lanes and wavefronts: 162, J = 170).

The forward pass's mean and rstd are compared with the definition; everything else with the formulas evaluated at the mean
and rstd that were stored, which is what the kernels read, so that an offset of the data does not widen a bound:

  mean   sums: H u max|x|; joins m + d f (d <= 2 max|x|, f within 3u): 8 u max|x| each, J of them
  rstd   squares and their sum (H + 4) u, joins 8 u each, half of it for the root; the mean's error enters squared; root,
         division and eps 4 u
  xh     (x - m) r: 2u |xh|
  p      xh gamma + beta: ep = u (3 |xh gamma| + |p|)
  sigmoid  es = s (1 - s) (1.25 |p| + 2) u + 3 s u: -p log2(e) rounded (u, its constant u / 4), 2^t 2u, 1 + t u, 1 / t 2u
  y      none 0, leaky u |y|, SiLU |p| es + u |y|;  |f'| <= 1.1 (or the slope) times ep
  f'     none, leaky: exact, but for |p| <= ep, where either slope may be taken;  SiLU s + p s (1 - s):
         (1 + |p|) es + 3u (|p| s (1 - s) + s), and |f''| <= 1/2 times ep
  dp     dy f': |dy| times the error of f', u |dp|
  sums   the terms' errors and H u times the sum of their magnitudes
  dx     r (gamma dp - s1 - xh s2): the errors of its parts and 4u of their magnitudes
Rounding to zero below 2^-126 is covered by `tiny` per term."""
import numpy as np

U = 2.0 ** -24
H, J = 400, 170
TINY = 2.0 ** -125


def rows_of(a, N, C, HW, G, last):
    """x-shaped data as (N, G, channels of a group, pixels), 64 bits."""
    a = np.asarray(a, np.float64)
    a = a.reshape(N, HW, C).transpose(0, 2, 1) if last else a.reshape(N, C, HW)
    return a.reshape(N, G, C // G, HW)


def back(a, N, C, HW, last):
    a = a.reshape(N, C, HW)
    return np.ascontiguousarray(a.transpose(0, 2, 1)) if last else a


def _per_channel(v, G, C, default):
    v = np.full(C, default) if v is None else np.asarray(v, np.float64)
    return v.reshape(1, G, C // G, 1)


def _sigmoid(p):
    with np.errstate(over='ignore'):
        s = 1 / (1 + np.exp(-p))
    return s, (s * (1 - s) * (1.25 * np.abs(p) + 2) + 3 * s) * U


def statistics(x, N, C, HW, G, last, eps):
    """(mean, rstd) of the definition, (N * G,), and the bounds of their errors."""
    r = rows_of(x, N, C, HW, G, last)
    mean = r.mean((2, 3))
    var = ((r - mean[:, :, None, None]) ** 2).mean((2, 3))
    top = np.abs(r).max((2, 3))
    dm = (H + 8 * J) * U * top
    rstd = 1 / np.sqrt(var + eps)
    rel = ((H + 8 * J) / 2 + 8) * U + 0.5 * (dm * rstd) ** 2
    return mean.reshape(-1), rstd.reshape(-1), dm.reshape(-1) + TINY, (rel * rstd).reshape(-1)


class Pass:
    """The parts that forward and backward share: xh, p and its error, at a given mean and rstd (N * G,)."""

    def __init__(self, x, gamma, beta, mean, rstd, N, C, HW, G, last, act, slope):
        self.dims, self.act, self.slope = (N, C, HW, last), act, slope
        self.ga, be = _per_channel(gamma, G, C, 1.0), _per_channel(beta, G, C, 0.0)
        m, self.r = (np.asarray(v, np.float64).reshape(N, G, 1, 1) for v in (mean, rstd))
        self.xh = (rows_of(x, N, C, HW, G, last) - m) * self.r
        self.p = self.xh * self.ga + be
        self.ep = U * (3 * np.abs(self.xh * self.ga) + np.abs(self.p)) + TINY
        self.G = G

    def forward(self):
        """y and its bound."""
        p = self.p
        if self.act == 'silu':
            s, es = _sigmoid(p)
            y, err = p * s, np.abs(p) * es + 1.1 * self.ep
        elif self.act == 'leaky_relu':
            y, err = np.where(p >= 0, p, self.slope * p), max(1.0, abs(self.slope)) * self.ep
        else:
            y, err = p, self.ep
        return tuple(back(v, *self.dims) for v in (y, err + U * np.abs(y) + TINY))

    def backward(self, dy):
        """(dx, dgamma, dbeta) and their bounds."""
        N, C, HW, last = self.dims
        dy, p, xh, ga, r = rows_of(dy, N, C, HW, self.G, last), self.p, self.xh, self.ga, self.r
        if self.act == 'silu':
            s, es = _sigmoid(p)
            f = s + p * s * (1 - s)
            ef = (1 + np.abs(p)) * es + 3 * U * (np.abs(p) * s * (1 - s) + s) + 0.5 * self.ep
        elif self.act == 'leaky_relu':
            f, ef = np.where(p >= 0, 1.0, self.slope), np.where(np.abs(p) <= self.ep, abs(1 - self.slope), 0.0)
        else:
            f, ef = np.ones_like(p), 0.0
        dp = dy * f
        e_dp = np.abs(dy) * ef + U * np.abs(dp) + TINY

        def summed(v, e, axes, keep=False):
            return v.sum(axes, keepdims=keep), e.sum(axes, keepdims=keep) + H * U * np.abs(v).sum(axes, keepdims=keep)
        dbeta, e_dbeta = summed(dp, e_dp, (0, 3))
        t = dp * xh
        e_t = e_dp * np.abs(xh) + 3 * U * np.abs(t) + TINY
        dgamma, e_dgamma = summed(t, e_t, (0, 3))
        D = C // self.G * HW
        g, e_g = dp * ga, e_dp * np.abs(ga) + U * np.abs(dp * ga)
        s1, e_s1 = (v / D for v in summed(g, e_g, (2, 3), True))
        s2, e_s2 = (v / D for v in summed(t * ga, e_t * np.abs(ga) + U * np.abs(t * ga), (2, 3), True))
        e_s1, e_s2 = e_s1 + 2 * U * np.abs(s1), e_s2 + 2 * U * np.abs(s2)
        dx = r * (g - s1 - xh * s2)
        parts = np.abs(g) + np.abs(s1) + np.abs(xh * s2)
        e_dx = r * (e_g + e_s1 + np.abs(xh) * e_s2 + 4 * U * parts) + U * np.abs(dx) + TINY
        return ((back(dx, *self.dims), dgamma.reshape(-1), dbeta.reshape(-1)),
                (back(e_dx, *self.dims), e_dgamma.reshape(-1), e_dbeta.reshape(-1)))


def telling(refs, bounds):
    """Whether the bounds tell a result from zeros: for each output, at the element that is largest."""
    return [float(b.reshape(-1)[np.abs(r).argmax()]) < 0.02 * float(np.abs(r).max()) for r, b in zip(refs, bounds)]
