"""Sizes that the library's 32-bit extents cannot hold are refused, not taken modulo 2^32; groups are whole numbers."""
import numpy as np
import pytest

from litenn_amd.core.hip import api


@pytest.mark.parametrize('extents', [(1, 1, (1 << 32) + 64, 1), (1 << 32, 8, 4, 2), (2, (1 << 32) + 8, 4, 2), (1, 8, 4, (1 << 32) + 2),
                                     (1, 8, -(1 << 32) + 4, 2), (1, 8, 1 << 31, 2)])
def test_descriptor_extents(extents):
    with pytest.raises(api.HipException) as e:
        api.group_norm_desc(*extents)
    assert e.value.code == api.ERR_UNSUPPORTED


def test_descriptor_keeps_what_fits():
    d = api.group_norm_desc((1 << 31) - 1, -1, 4, 2)      # the library judges it
    assert (d.N, d.C) == ((1 << 31) - 1, -1)


@pytest.mark.parametrize('extents', [(1 << 32 | 1, 4, 4, 4), (1, 1 << 32 | 4, 4, 4), (1, 4, 1 << 32 | 4, 4), (1, 4, 4, 1 << 32 | 4), (1, 4, 1 << 31, 4)])
def test_weight_gradient_extents(extents):
    with pytest.raises(api.HipException) as e:
        api.gemm_wgrad8(0, *extents, 8, 8, 8)             # before any pointer is looked at
    assert e.value.code == api.ERR_UNSUPPORTED


def test_through_tensors(nn_backend):
    """A tensor of 2^32 + 64 elements (nothing is allocated before the first read): its last 64 must not stand for all."""
    nn = nn_backend
    x_t = nn.Tensor((1, 1, (1 << 32) + 64))
    for last, t in ((False, x_t), (True, nn.Tensor((1, (1 << 32) + 64, 1)))):
        with pytest.raises(api.HipException) as e:
            nn.group_norm(t, 1, channels_last=last)
        assert e.value.code == api.ERR_UNSUPPORTED
    assert not x_t._get_buffers()[0].has_ptr()
    small_t = nn.Tensor_from_value(np.ones((2, 5), np.float32))
    for groups in (2.5, 0.5, 1.0000001):
        with pytest.raises(ValueError, match='groups'):
            nn.group_norm(small_t, groups)
