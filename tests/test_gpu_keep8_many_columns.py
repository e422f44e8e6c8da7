"""The weight gradient from a kept input with more columns than one launch lays out: whole numbers, exact; and its scratch."""
import numpy as np
import pytest

from oracle.keep8 import keep8_encode, keep8_pack
from tests.gpu_util import DevArr, say
from tests.test_gpu_keep8 import wgrad

pytestmark = pytest.mark.gpu
RUN = 1 << 22


@pytest.mark.parametrize('shape', [(1, 2, 3, RUN + 5), (1, 2, RUN + 260, 3), (2, 1, 2, RUN + 9), (2, 1, RUN + 3, 2), (1, 40, 1, RUN + 1),
                                   (1, 3, 2, RUN), (1, 33, RUN + 4, 1)])
def test_runs_of_columns(hip, shape):
    batch, rows, K, M = shape
    say(f'wgrad8 many columns {shape}')
    rs = np.random.RandomState(50)
    x = rs.randint(-3, 4, (batch, rows, K)).astype(np.float32)
    dy = rs.randint(-4, 5, (batch, rows, M)).astype(np.float32)
    ref = np.matmul(x.transpose(0, 2, 1), dy)           # small whole numbers: exact in fp32
    assert np.array_equal(wgrad(hip, x, dy), ref)
    assert np.array_equal(wgrad(hip, x, dy, prefill=3.0), ref + 3)


def test_scratch_stays_bounded(hip):
    """One row, 2^24 columns: laid out at once, its 32-row fragments would take 3.2 GB."""
    say('wgrad8 scratch')
    hip.release_device(0)                                # lets go of scratch that earlier calls grew
    M = 1 << 24
    x, dy = np.ones((1, 1, 1), np.float32), np.arange(M, dtype=np.float32).reshape(1, 1, M)
    X8 = DevArr(hip, np.concatenate([keep8_pack(*keep8_encode(x)), np.zeros(3, np.uint8)]).view(np.float32))
    dY, dW = DevArr(hip, dy), DevArr(hip, shape=(M,), fill=0.0)
    hip.synchronize(0)
    before = hip.mem_info(0)[0]
    hip.gemm_wgrad8(0, 1, 1, 1, M, X8.ptr, dY.ptr, dW.ptr, 0)
    hip.synchronize(0)
    # a gigabyte at most, and a quarter of it on top, as scratch grows
    assert before - hip.mem_info(0)[0] <= 1.26 * 2 ** 30
    assert np.array_equal(dW.get(), dy.reshape(-1))
    hip.release_device(0)
