"""The weight gradient from a kept input where dO is next to the end of the fp32 range.  dO goes to the matrix pipe as three
bf16 numbers, and that pipe takes a bf16 input below 2^-126 for 0: the parts of dO that lie there are lost, less than
2^-126 (1 + 2^-7) of a value, and so are results below 2^-126.  With terms x dO over `rows` rows:
  |error| <= 2^-126 ((1 + 2^-7) sum |x| + rows + 1) + (3 rows + 4) u sum |x dO|
From |dO| = 2^-110 up nothing is lost: l, its last 8 bits, begins at 2^-126."""
import numpy as np
import pytest

from tests.gpu_util import say
from tests.test_gpu_keep8 import wgrad

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize('rows', [1, 40])
@pytest.mark.parametrize('scale', [0, -20, 40])
def test_small_gradients(hip, rows, scale):
    say(f'wgrad8 small gradients rows={rows} x scale 2^{scale}')
    rs = np.random.RandomState(60)
    x = np.ldexp(rs.randint(64, 128, (1, rows, 32)), scale).astype(np.float32)      # held exactly
    for low, high in ((-149, -126), (-135, -115), (-118, -105), (-110, -80)):
        dy = np.ldexp(rs.uniform(1, 2, (1, rows, 64)) * rs.choice([-1, 1], (1, rows, 64)), rs.randint(low, high, (1, rows, 64))).astype(np.float32)
        xt, d = x[0].T.astype(np.float64), dy[0].astype(np.float64)
        mag = np.abs(xt) @ np.abs(d)
        lost = 2.0 ** -126 * (rows + 1) + (0 if low >= -110 else 2.0 ** -126 * (1 + 2.0 ** -7) * xt.sum(1, keepdims=True))
        assert (np.abs(wgrad(hip, x, dy)[0] - xt @ d) <= lost + (3 * rows + 4) * U * mag).all(), (low, high)
