"""8-bit activation copies through the C ABI: bit-exact codes and values, and the weight gradient read from a copy."""
import numpy as np
import pytest

from oracle.keep8 import keep8_decode, keep8_encode, keep8_pack, keep8_values
from tests.gpu_util import DevArr, say

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def activations(seed, n):
    rs = np.random.RandomState(seed)
    x = rs.normal(0, 1, n) * np.repeat(np.exp2(rs.uniform(-40, 40, (n + 31) // 32)), 32)[:n]
    x[rs.uniform(size=n) < 0.1] = 0
    return x.astype(np.float32)


def round_trip(api, x, off=0):
    """(bytes of the copy, values read back); off: 4-byte steps the fp32 pointers, and bytes the copy, are moved by."""
    n = x.size
    X = DevArr(api, np.concatenate([np.zeros(off, np.float32), x]))
    K = DevArr(api, shape=((api.bytes8(n) + off + 3) // 4,), fill=np.float32(3.0))
    B = DevArr(api, shape=(n + off + 1,), fill=7.0)
    api.encode8(0, n, X.ptr + 4 * off, K.ptr + off)
    api.decode8(0, n, K.ptr + off, B.ptr + 4 * off)
    back = B.get()
    assert (back[:off] == 7.0).all() and back[off + n] == 7.0        # nothing around the result was touched
    return K.get().view(np.uint8)[off:off + api.bytes8(n)], back[off:off + n]


@pytest.mark.parametrize('n', [1, 2, 3, 4, 5, 31, 32, 33, 63, 64, 100, 1000, 4097, 100003, 1 << 20])
def test_round_trip(hip, n):
    for off in (0, 1):
        say(f'keep8 n={n} off={off}')
        x = activations(n, n)
        raw, back = round_trip(hip, x, off)
        codes, byte = keep8_encode(x)
        assert np.array_equal(raw, keep8_pack(codes, byte))
        assert np.array_equal(back, keep8_decode(codes, byte, n))


def test_edges(hip):
    fmax = np.finfo(np.float32).max
    rows = [[], [127.5], [np.nextafter(np.float32(127.5), np.float32(0))], [127, 2.5, 3.5, -2.5, 0.5, -0.5], [fmax, -fmax, fmax / 3],
            [1e-45, 2.0 ** -126], [2.0 ** -120, 1e-40], [np.nan, 1], [1, np.inf], [-np.inf], [-0.0, 0.0], [2.0 ** 121 * 127.5, 1e38], [-1e-30]]
    x = np.zeros((len(rows), 32), np.float32)
    for r, v in zip(x, rows):
        r[32 - len(v):] = np.array(v, np.float32)
    say('keep8 edges')
    raw, back = round_trip(hip, x.reshape(-1))
    codes, byte = keep8_encode(x)
    assert np.array_equal(raw, keep8_pack(codes, byte))
    assert np.array_equal(back, keep8_decode(codes, byte, x.size), equal_nan=True)


def test_refusals(hip):
    B = DevArr(hip, shape=(64,), fill=0.0)
    for call in (lambda: hip.encode8(0, 4, None, B.ptr), lambda: hip.decode8(0, 4, B.ptr, None), lambda: hip.gemm_wgrad8(0, 1, 1, 1, 1, None, B.ptr, B.ptr),
                 lambda: hip.gemm_wgrad8(0, 0, 1, 1, 1, B.ptr, B.ptr, B.ptr), lambda: hip.gemm_wgrad8(0, 1, 1, -1, 1, B.ptr, B.ptr, B.ptr)):
        with pytest.raises(hip.HipException) as e:
            call()
        assert e.value.code == hip.ERR_INVALID
    for call in (lambda: hip.encode8(0, 1 << 62, B.ptr, B.ptr), lambda: hip.decode8(0, 1 << 29, B.ptr, B.ptr),
                 lambda: hip.gemm_wgrad8(0, 1, 1 << 20, 1 << 10, 1, B.ptr, B.ptr, B.ptr)):
        with pytest.raises(hip.HipException) as e:
            call()
        assert e.value.code == hip.ERR_UNSUPPORTED
    hip.encode8(0, 0, None, None)      # nothing to do
    d = hip.group_norm_desc(1, 4, 4, 2)
    p = B.ptr
    for call in (lambda: hip.group_norm_fwd(0, hip.group_norm_desc(1, 4, 4, 3), p, p, p, p, p, p),
                 lambda: hip.group_norm_fwd(0, hip.group_norm_desc(0, 4, 4, 2), p, p, p, p, p, p),
                 lambda: hip.group_norm_fwd(0, hip.group_norm_desc(1, 4, 4, 2, eps=0.0), p, p, p, p, p, p),
                 lambda: hip.group_norm_fwd(0, hip.group_norm_desc(1, 4, 4, 2, eps=float('nan')), p, p, p, p, p, p),
                 lambda: hip.group_norm_fwd(0, hip.group_norm_desc(1, 4, 4, 2, act=7), p, p, p, p, p, p),
                 lambda: hip.group_norm_fwd(0, d, None, p, p, p, p, p), lambda: hip.group_norm_fwd(0, d, p, p, p, p, None, p),
                 lambda: hip.group_norm_bwd(0, d, p, p, p, p, p, p, p, p, p, p), lambda: hip.group_norm_bwd(0, d, None, None, p, p, p, p, p, p, p, p),
                 lambda: hip.group_norm_bwd(0, d, p, None, p, p, p, p, None, p, p, p)):
        with pytest.raises(hip.HipException) as e:
            call()
        assert e.value.code == hip.ERR_INVALID
    with pytest.raises(hip.HipException) as e:
        hip.group_norm_fwd(0, hip.group_norm_desc(1 << 15, 1 << 10, 1 << 10, 2), p, p, p, p, p, p)
    assert e.value.code == hip.ERR_UNSUPPORTED
    hip.synchronize(0)


def wgrad(api, x, dy, prefill=None, off=0):
    """dW of x (batch, rows, K) kept in 8 bits and dy (batch, rows, M)."""
    batch, rows, K = x.shape
    M = dy.shape[2]
    raw = keep8_pack(*keep8_encode(x))
    raw = np.concatenate([np.zeros(off, np.uint8), raw, np.zeros(-(raw.size + off) % 4, np.uint8)])
    X8 = DevArr(api, raw.view(np.float32))
    dY = DevArr(api, np.concatenate([np.zeros(off, np.float32), dy.reshape(-1)]))
    dW = DevArr(api, shape=(off + batch * K * M + 1,), fill=np.nan if prefill is None else prefill)
    api.gemm_wgrad8(0, batch, rows, K, M, X8.ptr + off, dY.ptr + 4 * off, dW.ptr + 4 * off, 0 if prefill is None else 1)
    got = dW.get()
    edge = np.concatenate([got[:off], got[off + batch * K * M:]])
    assert np.isnan(edge).all() if prefill is None else (edge == prefill).all()
    return got[off:off + batch * K * M].reshape(batch, K, M)


SHAPES = [  # batch, rows, K, M
    (1, 1, 1, 1), (1, 1, 5, 3), (1, 3, 33, 17), (1, 32, 64, 64), (1, 33, 65, 31), (2, 40, 24, 56), (3, 7, 130, 66), (1, 1000, 333, 129),
    (1, 257, 256, 256), (1, 64, 300, 520), (1, 4096, 16, 24), (1, 9000, 128, 128), (5, 100, 32, 32), (1, 31, 1024, 96), (1, 513, 260, 700),
    (1, 20000, 3, 5), (70, 2, 4, 4), (1, 300, 1, 1000), (1, 300, 1000, 1), (1, 512, 512, 512), (1, 2048, 768, 640)]


@pytest.mark.parametrize('shape', SHAPES)
def test_wgrad_integer_exact(hip, shape):
    """Whole numbers that the copy holds exactly and whose products and sums stay below 2^24: any right order of addition
    gives the same bits."""
    batch, rows, K, M = shape
    say(f'wgrad8 {shape}')
    rs = np.random.RandomState(11)
    x = rs.randint(-15, 16, (batch, rows, K)).astype(np.float32)
    dy = rs.randint(-8, 9, (batch, rows, M)).astype(np.float32)
    assert np.array_equal(keep8_values(x), x)
    ref = np.matmul(x.transpose(0, 2, 1).astype(np.float64), dy.astype(np.float64))
    assert np.array_equal(wgrad(hip, x, dy), ref)
    assert np.array_equal(wgrad(hip, x, dy, prefill=3.0), ref + 3)
    assert np.array_equal(wgrad(hip, x, dy, off=1), ref)


@pytest.mark.parametrize('shape', SHAPES)
def test_wgrad_float(hip, shape):
    """rows products, their sum formed from at most 3 rows fp32 additions:  |error| <= (3 rows + 4) u sum |x dy|."""
    batch, rows, K, M = shape
    say(f'wgrad8 float {shape}')
    rs = np.random.RandomState(12)
    x = (activations(13, batch * rows * K).reshape(batch, rows, K) if rows < 100 else rs.normal(0, 1, (batch, rows, K))).astype(np.float32)
    dy = (rs.normal(0, 1, (batch, rows, M)) * np.exp2(rs.uniform(-20, 20, (batch, rows, 1)))).astype(np.float32)
    v = keep8_values(x).astype(np.float64).transpose(0, 2, 1)
    ref, mag = np.matmul(v, dy.astype(np.float64)), np.matmul(np.abs(v), np.abs(dy).astype(np.float64))
    assert (np.abs(wgrad(hip, x, dy) - ref) <= (3 * rows + 4) * U * mag + 2.0 ** -140).all()


def test_wgrad_one_row_keeps_all_bits_of_the_gradient(hip):
    """One row: a single product per output, so no digit of dO may be lost on the way - including huge, tiny and
    infinite ones."""
    say('wgrad8 one row')
    rs = np.random.RandomState(14)
    x = rs.randint(1, 128, (1, 1, 40)).astype(np.float32)
    dy = (rs.normal(0, 1, (1, 1, 600)) * np.exp2(rs.uniform(-100, 100, (1, 1, 600)))).astype(np.float32)
    got = wgrad(hip, x, dy)
    ref = np.matmul(x.transpose(0, 2, 1).astype(np.float64), dy.astype(np.float64))
    assert (np.abs(got - ref) <= 3 * U * np.abs(ref)).all()
    dy[0, 0, :6] = [np.inf, -np.inf, np.nan, 3e38, -3e38, 1e-38]
    got = wgrad(hip, x, dy)
    with np.errstate(over='ignore', invalid='ignore'):
        ref = np.matmul(x.transpose(0, 2, 1).astype(np.float64), dy.astype(np.float64)).astype(np.float32)
    assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(np.isinf(got), np.isinf(ref))
    assert np.array_equal(np.sign(got[np.isinf(got)]), np.sign(ref[np.isinf(ref)]))


def test_wgrad_nonfinite_stays_in_its_place(hip):
    """A NaN in x reaches its block's columns only, one in dO its column only."""
    say('wgrad8 nonfinite')
    rs = np.random.RandomState(15)
    x, dy = rs.normal(0, 1, (1, 70, 96)).astype(np.float32), rs.normal(0, 1, (1, 70, 40)).astype(np.float32)
    x[0, 9, 40] = np.nan
    dy[0, 50, 7] = np.inf
    got = wgrad(hip, x, dy)[0]
    bad = ~np.isfinite(got)
    want = np.zeros((96, 40), bool)
    want[32:64, :] = True
    want[:, 7] = True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize('shape', [(20000, 2, 3, 2), (1, 600000, 2, 3)])
def test_wgrad_in_parts(hip, shape):
    """More batch items, and more rows, than one launch lays out: whole numbers, exact, written and accumulated."""
    say(f'wgrad8 in parts {shape}')
    batch, rows, K, M = shape
    rs = np.random.RandomState(16)
    x = rs.randint(-3, 4, (batch, rows, K)).astype(np.float32)
    dy = rs.randint(-4, 5, (batch, rows, M)).astype(np.float32)
    ref = np.matmul(x.transpose(0, 2, 1).astype(np.float64), dy.astype(np.float64))     # below 600000 * 12 < 2^24
    assert np.array_equal(wgrad(hip, x, dy), ref)
    assert np.array_equal(wgrad(hip, x, dy, prefill=3.0), ref + 3)
