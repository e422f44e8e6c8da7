"""Activations kept in 8 bits, restated from the format's definition (no reference file: the reference keeps fp32)."""
import numpy as np


def keep8_encode(x):
    """(codes int8 (blocks, 32), exponent bytes uint8 (blocks,)) of the flat values of x."""
    x = np.asarray(x, np.float32).reshape(-1).astype(np.float64)
    v = np.concatenate([x, np.zeros(-x.size % 32)]).reshape(-1, 32)
    bad = ~np.isfinite(v).all(1)
    a = np.where(bad, 0.0, np.abs(np.where(np.isfinite(v), v, 0.0)).max(1))
    # the smallest e of [-126, 121] with a 2^-e < 127.5 (ldexp is exact; 121 whatever a)
    e = np.full(a.shape, 121)
    for t in range(120, -127, -1):
        e = np.where(np.ldexp(a, -t) < 127.5, t, e)
    with np.errstate(invalid='ignore'):
        q = np.clip(np.rint(np.ldexp(v, -e[:, None])), -127, 127)
    q = np.where(bad[:, None], 0, q)
    byte = np.where(bad, 255, np.where(a == 0, 0, e + 127))
    return q.astype(np.int8), byte.astype(np.uint8)


def keep8_decode(codes, byte, n):
    """The n float32 values that codes and exponent bytes stand for."""
    b = byte.astype(np.int64)
    v = np.ldexp(codes.astype(np.float64), np.where(b == 255, 0, b - 127)[:, None])
    v[b == 255] = np.nan
    return v.reshape(-1)[:n].astype(np.float32)


def keep8_pack(codes, byte):
    """The bytes of a copy as they lie in memory."""
    return np.concatenate([codes.reshape(-1).view(np.uint8), byte])


def keep8_values(x):
    """x after being kept in 8 bits and read back, in its shape."""
    x = np.asarray(x, np.float32)
    return keep8_decode(*keep8_encode(x), x.size).reshape(x.shape)
