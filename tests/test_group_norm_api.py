"""nn.group_norm, nn.GroupNorm and nn.keep8 through the Python layer: on the numpy stand-in (host logic) and - marked gpu - on
the real library."""
import itertools

import numpy as np
import pytest

from oracle import conv2d_dw, conv2d_dx, conv2d_fwd
from oracle.group_norm import group_norm_bwd, group_norm_fwd
from oracle.keep8 import keep8_decode, keep8_encode, keep8_pack, keep8_values

ACTS = {0: 'none', 1: 'leaky_relu', 2: 'silu'}


class FakeNorm:
    """The stand-in's versions of the calls: its memory, the oracle's arithmetic."""

    def __init__(self, fake):
        self.fake, self.calls = fake, []

    def _bytes(self, ptr):
        return self.fake.mem[ptr].view(np.uint8)

    def _kept(self, ptr, n):
        b = self._bytes(ptr)
        blocks = -(-n // 32)
        return keep8_decode(b[:32 * blocks].view(np.int8).reshape(-1, 32), b[32 * blocks:33 * blocks], n)

    def encode8(self, dev, n, src, dst):
        self.calls.append('encode8')
        raw = keep8_pack(*keep8_encode(self.fake.f(src)[:n]))
        self._bytes(dst)[:raw.size] = raw

    def decode8(self, dev, n, src, dst):
        self.calls.append('decode8')
        self.fake.f(dst)[:n] = self._kept(src, n)

    def gemm_wgrad8(self, dev, batch, rows, K, M, x8, dO, dW, beta=0):
        self.calls.append('gemm_wgrad8')
        x = self._kept(x8, batch * rows * K).reshape(batch, rows, K).astype(np.float64)
        r = np.matmul(x.transpose(0, 2, 1), self.fake.f(dO, (batch, rows, M)).astype(np.float64))
        self.fake._put(self.fake.f(dW, (batch, K, M)), r, beta)

    def _args(self, d, gamma, beta):
        return ((None if gamma is None else self.fake.f(gamma)[:d.C]), (None if beta is None else self.fake.f(beta)[:d.C]),
                (d.N, d.C, d.HW, d.groups, bool(d.channels_last), ACTS[d.act], d.slope))

    def group_norm_fwd(self, dev, d, x, gamma, beta, y, mean, rstd, x8=None):
        self.calls.append('group_norm_fwd')
        n = d.N * d.C * d.HW
        xv = self.fake.f(x)[:n]
        ga, be, rest = self._args(d, gamma, beta)
        ry, rm, rr = group_norm_fwd(xv, ga, be, *rest, d.eps)
        for ptr, v in ((y, ry), (mean, rm), (rstd, rr)):
            self.fake.f(ptr)[:v.size] = v.reshape(-1)
        if x8 is not None:
            raw = keep8_pack(*keep8_encode(xv))
            self._bytes(x8)[:raw.size] = raw

    def group_norm_bwd(self, dev, d, x, x8, gamma, beta, mean, rstd, dy, dx, dgamma, dbeta, beta_dx=0, beta_dgamma=0, beta_dbeta=0):
        assert (x is None) != (x8 is None)
        self.calls.append('group_norm_bwd8' if x is None else 'group_norm_bwd')
        n, rows = d.N * d.C * d.HW, (d.N, d.groups)
        ga, be, rest = self._args(d, gamma, beta)
        xv = self.fake.f(x)[:n] if x is not None else self._kept(x8, n)
        r = group_norm_bwd(xv, self.fake.f(dy)[:n], ga, be, self.fake.f(mean, rows), self.fake.f(rstd, rows), *rest)
        for ptr, v, b in zip((dx, dgamma, dbeta), r, (beta_dx, beta_dgamma, beta_dbeta)):
            if ptr is not None:
                self.fake._put(self.fake.f(ptr)[:v.size], v.reshape(-1), b)


@pytest.fixture
def nn8(nn_backend, monkeypatch):
    nn = nn_backend
    nn._test_norm = None
    if nn._test_fake is not None:
        from litenn_amd.core.hip import api
        nn._test_norm = f = FakeNorm(nn._test_fake)
        for name in ('encode8', 'decode8', 'gemm_wgrad8', 'group_norm_fwd', 'group_norm_bwd'):
            monkeypatch.setattr(api, name, getattr(f, name))
    yield nn
    nn._test_norm = None


def close(got, ref, tol=2e-5):
    """Normalised maximum error: everything here is some hundred terms of magnitude 1 added up in fp32, 2e-5 = 330 u."""
    assert got.shape == ref.shape
    assert np.abs(got - ref).max() <= tol * max(1.0, np.abs(ref).max()), np.abs(got - ref).max()


def lay(x, last):
    return np.ascontiguousarray(np.moveaxis(x, 1, -1)) if last else x


@pytest.mark.parametrize('keep', ['', 'fused', 'after'])
@pytest.mark.parametrize('last', [False, True])
def test_group_norm(nn8, last, keep):
    nn = nn8
    rs = np.random.RandomState(1)
    for shape, groups in (((2, 6, 5, 7), 3), ((5, 16), 4), ((3, 8, 4), 1), ((1, 4, 2, 3, 3), 2)):
        N, C = shape[:2]
        HW = int(np.prod(shape)) // (N * C)
        for act, alpha in (('silu', 0.0), (None, 0.0)):
            x, dy = lay(rs.normal(0.5, 2, shape).astype(np.float32), last), lay(rs.normal(0, 1, shape).astype(np.float32), last)
            ga, be = rs.normal(1, 0.3, C).astype(np.float32), rs.normal(0, 0.3, C).astype(np.float32)
            x_t, ga_t, be_t = (nn.Tensor_from_value(v) for v in (x, ga, be))
            y_t = nn.group_norm(x_t, groups, ga_t, be_t, 1e-3, act, channels_last=last, keep8=keep == 'fused')
            if keep == 'after':
                nn.keep8(x_t)
            x_t.get_grad().fill(1.0)
            be_t.get_grad().fill(2.0)
            nn.backward({y_t: dy}, grad_for_non_trainables=True)
            xs = keep8_values(x) if keep else x
            ry, mean, rstd = group_norm_fwd(x, ga, be, N, C, HW, groups, last, act or 'none', alpha, 1e-3)
            dx, dg, db = group_norm_bwd(xs, dy, ga, be, mean, rstd, N, C, HW, groups, last, act or 'none', alpha)
            close(y_t.np().reshape(ry.shape), ry)
            close(x_t.get_grad().np().reshape(dx.shape), dx + 1)
            close(ga_t.get_grad().np(), dg)
            close(be_t.get_grad().np(), db + 2)
            if keep:
                assert not x_t._get_buffers()[0].has_ptr()
                assert np.array_equal(x_t.np(), keep8_values(x))
            if nn._test_norm is not None:
                assert nn._test_norm.calls.count('group_norm_bwd8' if keep else 'group_norm_bwd') == 1   # one pass for all three
                assert nn._test_norm.calls.count('decode8') == (1 if keep else 0)                        # by np() alone
                nn._test_norm.calls.clear()


def test_activations_and_defaults(nn8):
    nn = nn8
    rs = np.random.RandomState(2)
    x = rs.normal(0, 1, (3, 8, 10)).astype(np.float32)
    for kw, name, slope in ((dict(activation='relu'), 'leaky_relu', 0.0), (dict(activation='leaky_relu', alpha=0.3), 'leaky_relu', 0.3),
                            (dict(activation='leaky_relu'), 'leaky_relu', 0.1), (dict(), 'none', 0.0)):
        y = nn.group_norm(nn.Tensor_from_value(x), 2, **kw)
        close(y.np(), group_norm_fwd(x, None, None, 3, 8, 10, 2, False, name, slope, 1e-5)[0])


def test_only_wanted_gradients(nn8):
    nn = nn8
    x = np.random.RandomState(3).normal(0, 1, (2, 4, 6)).astype(np.float32)
    ga_t, be_t = nn.Tensor_from_value(np.ones(4, np.float32)), nn.Tensor_from_value(np.zeros(4, np.float32))
    opt = nn.optimizer.SGD([ga_t], lr=0.1)
    x_t = nn.Tensor_from_value(x)
    y_t = nn.group_norm(x_t, 2, ga_t, be_t)
    y_t.backward()
    assert ga_t.has_grad() and not x_t.has_grad() and not be_t.has_grad()
    g = ga_t.get_grad().np()
    close(g, group_norm_bwd(x, np.ones_like(x), None, None, *group_norm_fwd(x, None, None, 2, 4, 6, 2, False, 'none', 0, 1e-5)[1:],
                            2, 4, 6, 2, False, 'none', 0)[1])
    with nn.optimizer.freeze():
        y_t = nn.group_norm(x_t, 2, ga_t, be_t)
    y_t.backward(grad_for_non_trainables=True)
    assert np.array_equal(ga_t.get_grad().np(), g) and x_t.has_grad() and be_t.has_grad()
    del opt


def test_one_tensor_in_two_places(nn8):
    """gamma and beta the same tensor, and x a view of it as well."""
    nn = nn8
    v = np.array([1.0, 2.0, -0.5, 0.25], np.float32)
    v_t = nn.Tensor_from_value(v)
    y_t = nn.group_norm(v_t.reshape((1, 4)), 1, v_t, v_t)
    dy = np.array([[0.5, -1, 2, 0.25]], np.float32)
    nn.backward({y_t: dy}, grad_for_non_trainables=True)
    _, mean, rstd = group_norm_fwd(v, v, v, 1, 4, 1, 1, False, 'none', 0, 1e-5)
    dx, dg, db = group_norm_bwd(v, dy, v, v, mean, rstd, 1, 4, 1, 1, False, 'none', 0)
    close(v_t.get_grad().np(), dx.reshape(-1) + dg + db)


def test_two_backward_passes(nn8):
    """A second sweep forms its gradients again instead of taking the first one's for done."""
    nn = nn8
    x = np.random.RandomState(4).normal(0, 1, (2, 4, 6)).astype(np.float32)
    x_t = nn.Tensor_from_value(x)
    y_t = nn.group_norm(x_t, 2, activation='silu')
    dy = np.random.RandomState(5).normal(0, 1, x.shape).astype(np.float32)
    nn.backward({y_t: dy}, grad_for_non_trainables=True)
    one = x_t.get_grad().np()
    y_t.free_grad()
    nn.backward({y_t: dy}, grad_for_non_trainables=True)
    close(x_t.get_grad().np(), 2 * one)


def test_refusals(nn8):
    nn = nn8
    x_t = nn.Tensor_from_value(np.ones((2, 6, 3), np.float32))
    w_t = nn.Tensor_from_value(np.ones(6, np.float32))
    for call in (lambda: nn.group_norm(x_t, 4), lambda: nn.group_norm(x_t, 0), lambda: nn.group_norm(x_t, 2, eps=0.0),
                 lambda: nn.group_norm(x_t, 3, w_t.reshape((2, 3))), lambda: nn.group_norm(x_t, 3, channels_last=True, gamma_t=w_t),
                 lambda: nn.group_norm(w_t, 2), lambda: nn.group_norm(x_t, 2, activation='tanh'), lambda: nn.GroupNorm(4, 6),
                 lambda: nn.keep8(np.ones(3)), lambda: nn.keep8(x_t.get_grad())):
        with pytest.raises(ValueError):
            call()
    layer = nn.GroupNorm(2, 6)
    opt = nn.optimizer.SGD([w_t])
    for call in (lambda: nn.keep8(w_t), lambda: nn.keep8(layer.gamma), lambda: nn.keep8(layer.gamma.reshape((2, 3))),
                 lambda: nn.group_norm(w_t.reshape((1, 6)), 2, keep8=True)):
        with pytest.raises(ValueError, match='keep8'):
            call()
    assert np.array_equal(w_t.np(), np.ones(6))
    del opt


def test_keep8_state(nn8):
    """What ends, what survives and what frees the 8-bit state."""
    nn = nn8
    from litenn_amd.core.hip import HipBuffer
    rs = np.random.RandomState(6)
    x = rs.normal(0, 1, (10, 10)).astype(np.float32)
    kept = keep8_values(x)
    t = nn.Tensor_from_value(x)
    buf = t._get_buffers()[0]
    assert nn.keep8(t) is t and not buf.has_ptr() and buf.kept8() is not None
    assert np.array_equal(t.np(), kept)                      # a reader gets the decoded values ...
    assert buf.has_ptr() and buf.kept8() is not None
    nn.keep8(t)                                              # ... which go again without another rounding
    assert not buf.has_ptr() and np.array_equal(t.reshape((100,)).np(), kept.reshape(-1))
    c = t.copy()
    assert np.array_equal(c.np(), kept) and c._get_buffers()[0].kept8() is None
    t.set(x)                                                 # a write ends the state
    assert buf.kept8() is None and np.array_equal(t.np(), x)
    nn.keep8(t)
    t.fill(3.0)
    assert np.array_equal(t.np(), np.full((10, 10), 3.0, np.float32))
    t.set(x)
    nn.keep8(t)
    nn.core.op.add_const(t, 1.0, output_t=t)                 # reads the kept values, writes fp32
    close(t.np(), kept + 1)
    assert buf.kept8() is None
    fresh = nn.keep8(nn.Tensor((4, 4), init=nn.initializer.Scalar(2.0)))      # never touched before
    assert np.array_equal(fresh.np(), np.full((4, 4), 2.0, np.float32))
    with nn.devices._shallow_mode():
        nn.keep8(nn.group_norm(nn.Tensor((2, 4, 4)), 2, keep8=True))
    before = HipBuffer._object_count
    nn.keep8(nn.Tensor_from_value(x))
    assert HipBuffer._object_count == before                 # the copy goes with the tensor


def test_memory_of_a_kept_tensor(nn8):
    nn = nn8
    dev = nn.devices.get_current()[0]
    used = dev.get_used_memory()
    t = nn.Tensor_from_value(np.ones((64, 1000), np.float32))
    assert dev.get_used_memory() - used == 256000
    nn.keep8(t)
    assert dev.get_used_memory() - used == 66000
    del t
    assert dev.get_used_memory() == used


def _step(nn, x, w1, ga, be, w2, w3, b3, dy, keep):
    """conv - norm - SiLU - conv - dense, forward and backward; the gradients of all parameters and of x."""
    x_t, w1_t, ga_t, be_t, w2_t, w3_t, b3_t = (nn.Tensor_from_value(v) for v in (x, w1, ga, be, w2, w3, b3))
    h_t = nn.conv2D(x_t, w1_t)
    y_t = nn.group_norm(h_t, 4, ga_t, be_t, 1e-5, 'silu', keep8=keep)
    z_t = nn.conv2D(y_t, w2_t)
    f_t = z_t.reshape((z_t.shape[0], -1))
    o_t = nn.core.op.matmul_bias_act(f_t, w3_t, b3_t)
    if keep:
        nn.keep8(y_t)
        nn.keep8(f_t)
        assert all(not t._get_buffers()[0].has_ptr() for t in (h_t, y_t, z_t))
    nn.backward({o_t: dy}, grad_for_non_trainables=True)
    if keep:      # what was decoded on the way is gone again
        assert all(not t._get_buffers()[0].has_ptr() and t._get_buffers()[0].kept8() is not None for t in (h_t, y_t, z_t))
    return [o_t.np()] + [t.get_grad().np() for t in (x_t, w1_t, ga_t, be_t, w2_t, w3_t, b3_t)]


@pytest.mark.parametrize('keep', [False, True])
def test_training_pass(nn8, keep):
    nn = nn8
    rs = np.random.RandomState(7)
    x, dy = rs.normal(0, 1, (2, 3, 8, 8)).astype(np.float32), rs.normal(0, 1, (2, 5)).astype(np.float32)
    w1, w2 = rs.normal(0, 0.2, (8, 3, 3, 3)).astype(np.float32), rs.normal(0, 0.1, (4, 8, 3, 3)).astype(np.float32)
    ga, be = rs.normal(1, 0.2, 8).astype(np.float32), rs.normal(0, 0.2, 8).astype(np.float32)
    w3, b3 = rs.normal(0, 0.1, (256, 5)).astype(np.float32), rs.normal(0, 0.1, 5).astype(np.float32)
    got = _step(nn, x, w1, ga, be, w2, w3, b3, dy, keep)
    k = keep8_values if keep else lambda v: v
    h = np.asarray(conv2d_fwd(x, w1, 1, 1, 'same'), np.float32)
    y, mean, rstd = group_norm_fwd(h, ga, be, 2, 8, 64, 4, False, 'silu', 0, 1e-5)
    y = y.reshape(h.shape).astype(np.float32)
    z = np.asarray(conv2d_fwd(y, w2, 1, 1, 'same'), np.float32)
    f = z.reshape(2, -1)
    do = dy.astype(np.float64)
    dz = (do @ w3.T).reshape(z.shape)
    dyy = conv2d_dx(dz, w2, y.shape, 1, 1, 'same')
    dh, dg, db = group_norm_bwd(k(h), dyy, ga, be, mean, rstd, 2, 8, 64, 4, False, 'silu', 0)
    dh = dh.reshape(h.shape)
    ref = [f @ w3 + b3, conv2d_dx(dh, w1, x.shape, 1, 1, 'same'), conv2d_dw(x, dh, w1.shape, 1, 1, 'same'), dg, db,
           conv2d_dw(k(y), dz, w2.shape, 1, 1, 'same'), k(f).T @ do, do.sum(0)]
    if not keep:
        tols = [2e-5] * 8
    else:
        # the kernels' h, y and z differ from these in their last bits, so a value near the border between two codes may be
        # kept as its neighbour: one step, 2^-6 of its block's largest value, in one factor of a few of a gradient's terms
        tols = [2e-5] + [2e-3] * 6 + [2e-5]
    for g, r, tol in zip(got, ref, tols):
        close(g, np.asarray(r).reshape(g.shape), tol)


def test_layers_train(nn8):
    """Layers with the norm between them through an optimizer: every parameter moves, state round-trips."""
    nn = nn8

    class Net(nn.Module):
        def __init__(self):
            self.conv = nn.Conv2D(3, 8, 3)
            self.norm = nn.GroupNorm(2, 8, activation='leaky_relu', keep8=True)
            self.dense = nn.Dense(8 * 16, 6)
            self.norm2 = nn.GroupNorm(3, 6, channels_last=True, activation='silu')

        def forward(self, x):
            h = self.norm(self.conv(x))
            return self.norm2(self.dense(nn.flatten(h)))
    np.random.seed(1)
    net = Net()
    opt = nn.optimizer.Adam(net.trainables(), lr=1e-2)
    assert len(net.trainables()) == 8
    before = [t.np() for t in net.trainables()]
    x = np.random.RandomState(8).normal(0, 1, (4, 3, 4, 4)).astype(np.float32)
    for training in (True, False):
        net.set_training(training)
        opt.zero_grad()
        x_t = nn.Tensor_from_value(x)
        y = net(x_t)
        nn.square(y * nn.Tensor_from_value(np.arange(1, 7, dtype=np.float32).reshape(1, 6))).mean().backward()
        opt.step()
    if nn._test_norm is not None:
        assert nn._test_norm.calls.count('group_norm_bwd8') == 1      # only while training
    assert all(np.abs(t.np() - b).max() > 0 for t, b in zip(net.trainables(), before))
    state = net.dump_state()
    other = Net()
    other.load_state(state)
    assert np.array_equal(other(nn.Tensor_from_value(x)).np(), net(nn.Tensor_from_value(x)).np())


def test_dense_weight_gradient_reads_the_copy(nn8):
    nn = nn8
    rs = np.random.RandomState(9)
    for xs, ws in (((40, 24), (24, 16)), ((3, 10, 8), (3, 8, 12))):
        x, w = rs.normal(0, 1, xs).astype(np.float32), rs.normal(0, 1, ws).astype(np.float32)
        x_t, w_t = nn.Tensor_from_value(x), nn.Tensor_from_value(w)
        y_t = nn.matmul(x_t, w_t)
        nn.keep8(x_t)
        dy = rs.normal(0, 1, tuple(y_t.shape)).astype(np.float32)
        nn.backward({y_t: dy}, grad_for_non_trainables=True)
        close(w_t.get_grad().np(), np.matmul(np.swapaxes(keep8_values(x).astype(np.float64), -1, -2), dy))
        close(x_t.get_grad().np(), np.matmul(dy.astype(np.float64), np.swapaxes(w, -1, -2)))
        if nn._test_norm is not None:
            assert nn._test_norm.calls == ['encode8', 'gemm_wgrad8']
            nn._test_norm.calls.clear()


def test_other_gradients_decode(nn8):
    """square, mul and a convolution's kernel gradient on kept inputs."""
    nn = nn8
    rs = np.random.RandomState(10)
    x = rs.normal(0, 1, (2, 3, 6, 6)).astype(np.float32)
    a_t, b_t = nn.Tensor_from_value(x), nn.Tensor_from_value(x + 1)
    y_t = nn.square(a_t) + nn.mul(a_t, b_t)
    nn.keep8(a_t)
    nn.keep8(b_t)
    y_t.backward(grad_for_non_trainables=True)
    close(a_t.get_grad().np(), 2 * keep8_values(x) + keep8_values(x + 1))
    close(b_t.get_grad().np(), keep8_values(x))
    assert not a_t._get_buffers()[0].has_ptr() and not b_t._get_buffers()[0].has_ptr()


def test_descriptor_layout():
    import ctypes
    from litenn_amd.core.hip import api
    assert ctypes.sizeof(api.GroupNormDesc) == 32
    assert [api.bytes8(n) for n in (0, 1, 32, 33, 100003)] == [0, 33, 33, 66, 3126 * 33]
    with pytest.raises(api.HipException):
        api.bytes8(1 << 62)
    assert list(itertools.islice((f[0] for f in api.GroupNormDesc._fields_), 4)) == ['N', 'C', 'HW', 'groups']
