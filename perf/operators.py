"""The normalisation and 8-bit activation-checkpoint operators as a training or inference program calls them, with their
plain forms.

Five kinds of case:

  norm     group norm + activation, forward (inference)
  train    its forward and backward pass: y, dx, dgamma, dbeta
  train8   the same where the forward pass leaves x in 8 bits and the backward pass reads that copy instead of x
  keep8    an activation written in 8 bits and read back
  grad8    the weight gradient of a dense layer whose input was kept in 8 bits: dW = X8^T dO

8-bit copies: blocks of 32 elements in memory order share a power of two; int8 codes first (padded to whole blocks), then
one exponent byte per block (see include/litenn_hip.h)."""
import math

import torch

own = False

EPS = 1e-5
MOST = 1 << 26          # elements of the largest activation
MOST_MACS = 1 << 37     # multiply-adds of the largest weight gradient


# ---- cases ------------------------------------------------------------------
def listed():
    return [
        # one small image through an inference net: what counts is latency
        dict(name='norm first 1x64x14x14', kind='norm', N=1, C=64, HW=196, groups=8, last=False, act='leaky_relu'),
        # the activation behind the benchmark's 128-channel 56 x 56 convolution
        dict(name='norm first 32x128x56x56', kind='norm', N=32, C=128, HW=3136, groups=32, last=False, act='leaky_relu'),
        # a large channels-last batch, as a model whose 1x1 layers are dense layers holds it
        dict(name='norm last 16x128x128x256', kind='norm', N=16, C=256, HW=16384, groups=32, last=True, act='silu'),
        # training step of the layer above, channels first
        dict(name='train first 32x128x56x56', kind='train', N=32, C=128, HW=3136, groups=32, last=False, act='silu'),
        # odd everything: 37 x 41 images, 5 channels to a group
        dict(name='train last 3x37x41x60', kind='train', N=3, C=60, HW=1517, groups=12, last=True, act='silu'),
        # behind a dense layer: every row of (rows, 4096) is normalised by itself
        dict(name='train rows 8192x4096', kind='train', N=8192, C=4096, HW=1, groups=32, last=True, act='none'),
        # the same layers with the norm's input kept in 8 bits
        dict(name='train8 first 32x256x56x56', kind='train8', N=32, C=256, HW=3136, groups=32, last=False, act='silu'),
        dict(name='train8 last 8x64x64x320', kind='train8', N=8, C=320, HW=4096, groups=32, last=True, act='silu'),
        # a ragged activation, its last block not full, and a large one
        dict(name='keep8 100003', kind='keep8', n=100003),
        dict(name='keep8 64Mi', kind='keep8', n=1 << 26),
        # a ragged dense layer, and the 4096 -> 4096 layer at a training batch of rows
        dict(name='grad8 1000x333x129', kind='grad8', rows=1000, K=333, M=129),
        dict(name='grad8 8192x4096x4096', kind='grad8', rows=8192, K=4096, M=4096),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(['norm', 'train', 'train8', 'keep8', 'grad8'])
    if kind == 'keep8':
        return dict(kind=kind, n=_spread(rng, 1, MOST))
    if kind == 'grad8':
        while True:
            c = dict(kind=kind, rows=_spread(rng, 1, 16384), K=_spread(rng, 1, 4096), M=_spread(rng, 1, 4096))
            if c['rows'] * c['K'] * c['M'] <= MOST_MACS:
                return c
    most = MOST if kind == 'norm' else MOST // 2
    while True:
        groups, per = _spread(rng, 1, 32), _spread(rng, 1, 128)
        rows = rng.random() < 0.25      # behind a dense layer: no image
        c = dict(kind=kind, N=_spread(rng, 1, 16384 if rows else 64), C=groups * per,
                 HW=1 if rows else _spread(rng, 1, 256) * _spread(rng, 1, 256), groups=groups, last=rng.random() < 0.5,
                 act=rng.choice(['none', 'leaky_relu', 'silu'] if kind == 'norm' else ['none', 'silu']))
        # groups of one or two elements leave nothing of a gradient but rounding
        if per * c['HW'] >= 8 and c['N'] * c['C'] * c['HW'] <= most:
            return c


def work(case):
    """Reads and writes that the operator cannot do without: fp32 values 4 bytes, kept values 33/32 of a byte."""
    k = case['kind']
    if k == 'keep8':
        return dict(bytes=case['n'] * (4 + 4 + 2 * 33 / 32), flops=6 * case['n'])
    if k == 'grad8':
        r, K, M = case['rows'], case['K'], case['M']
        return dict(bytes=r * K * 33 / 32 + 4 * r * M + 4 * K * M, flops=2 * r * K * M)
    n = case['N'] * case['C'] * case['HW']
    few = 8 * case['C'] + 8 * case['N'] * case['groups']
    if k == 'norm':
        return dict(bytes=8 * n + few, flops=12 * n)
    if k == 'train':
        return dict(bytes=8 * n + 12 * n + 3 * few, flops=40 * n)
    return dict(bytes=8 * n + n * 33 / 32 + 8 * n + n * 33 / 32 + 3 * few, flops=50 * n)


# ---- inputs -----------------------------------------------------------------
def _values(case, seed):
    """The case's inputs, from the seed alone."""
    g = torch.Generator('cuda')
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device='cuda', dtype=torch.float32)
    k = case['kind']
    if k == 'keep8':
        # activations: some blocks far quieter than others, a tenth of the values zero
        x = normal(case['n'])
        x *= torch.exp(2 * normal(-(-case['n'] // 32))).repeat_interleave(32)[:case['n']]
        x[torch.rand(case['n'], generator=g, device='cuda') < 0.1] = 0
        return dict(x=x)
    if k == 'grad8':
        return dict(x=normal(case['rows'], case['K']), dy=normal(case['rows'], case['M']) * 1e-2)
    N, C, HW = case['N'], case['C'], case['HW']
    shape, per_c = ((N, HW, C), (1, 1, C)) if case['last'] else ((N, C, HW), (1, C, 1))
    x = normal(*shape)
    x *= torch.exp(0.5 * normal(*per_c))
    x += normal(*per_c)
    s = dict(x=x, gamma=1 + 0.2 * normal(C), beta=0.2 * normal(C))
    if k != 'norm':
        s['dy'] = normal(*shape)
    return s


def prepare(case, seed):
    s = _state(case, seed)
    torch.cuda.synchronize()      # see _own: the library's stream does not wait for torch's
    return s


def _state(case, seed):
    s = dict(case, **_values(case, seed))
    k = case['kind']
    if k == 'keep8':
        s['kept'] = torch.empty(-(-case['n'] // 32) * 33, dtype=torch.uint8, device='cuda')
        s['back'] = torch.empty_like(s['x'])
        return s
    if k == 'grad8':   # the backward pass has the kept input in hand, not the input
        s['kept'] = _pack(*_codes(s.pop('x').reshape(-1)))
        s['dW'] = torch.empty(case['K'], case['M'], device='cuda')
        return s
    # the buffers that a program's pool hands to the pass
    rows = case['N'] * case['groups']
    s.update(y=torch.empty_like(s['x']), mean=torch.empty(rows, device='cuda'), rstd=torch.empty(rows, device='cuda'))
    if k != 'norm':
        s.update(dx=torch.empty_like(s['x']), dgamma=torch.empty(case['C'], device='cuda'), dbeta=torch.empty(case['C'], device='cuda'))
    if k == 'train8':
        s['kept'] = torch.empty(-(-s['x'].numel() // 32) * 33, dtype=torch.uint8, device='cuda')
    return s


# ---- the framework's calls --------------------------------------------------
_ACTS = {'none': 0, 'leaky_relu': 1, 'silu': 2}
SLOPE = 0.1


def _own(s):
    """The calls on torch's memory.  The library queues its work on a stream of its own, and neither stream waits for the
    other: the inputs have to be written before the call (prepare waits for that), and a program that reads the outputs
    through torch, writes into the state or lets go of it waits for the device first (torch.cuda.synchronize(), or
    api.synchronize(0) for the library's stream alone).  Passes behind each other are in order."""
    from litenn_amd.core.hip import api
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    k = s['kind']
    if k == 'keep8':
        api.encode8(0, s['n'], p['x'], p['kept'])
        api.decode8(0, s['n'], p['kept'], p['back'])
        return s['back']
    if k == 'grad8':
        api.gemm_wgrad8(0, 1, s['rows'], s['K'], s['M'], p['kept'], p['dy'], p['dW'])
        return s['dW']
    d = api.group_norm_desc(s['N'], s['C'], s['HW'], s['groups'], s['last'], _ACTS[s['act']], SLOPE, EPS)
    api.group_norm_fwd(0, d, p['x'], p['gamma'], p['beta'], p['y'], p['mean'], p['rstd'], p.get('kept'))
    if k == 'norm':
        return s['y']
    api.group_norm_bwd(0, d, None if k == 'train8' else p['x'], p.get('kept'), p['gamma'], p['beta'], p['mean'], p['rstd'],
                       p['dy'], p['dx'], p['dgamma'], p['dbeta'])
    return s['y'], s['dx'], s['dgamma'], s['dbeta']


# ---- plain forms ------------------------------------------------------------
def _power(e):
    """2^e as float32, for whole e of [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _codes(x):
    """int8 codes (blocks, 32) and exponent bytes (blocks,) of a flat float32 tensor."""
    blocks = torch.nn.functional.pad(x, (0, -x.numel() % 32)).view(-1, 32)
    a = blocks.abs().amax(1)
    bad = ~torch.isfinite(a)
    m, k = torch.frexp(torch.where(bad, torch.zeros_like(a), a))      # a = m 2^k, 1/2 <= m < 1
    e = (k.to(torch.int32) - 7 + (m >= 127.5 / 128).to(torch.int32)).clamp(-126, 121)
    q = torch.round(blocks * _power(-e).unsqueeze(1)).clamp(-127, 127)
    byte = torch.where(bad, 255, torch.where(a == 0, 0, e + 127))
    return torch.where((bad | (a == 0)).unsqueeze(1), torch.zeros_like(q), q).to(torch.int8), byte.to(torch.uint8)


def _pack(q, byte):
    return torch.cat([q.view(torch.uint8).reshape(-1), byte])


def _kept_values(q, byte, n):
    """The float32 values that codes and exponent bytes stand for."""
    b = byte.to(torch.int32)
    scale = torch.where(b == 255, torch.full((), float('nan'), device=b.device), _power((b - 127).clamp(-126, 121)))
    return (q.to(torch.float32) * scale.unsqueeze(1)).reshape(-1)[:n]


def _act(p, name):
    if name == 'leaky_relu':
        return torch.where(p >= 0, p, SLOPE * p)
    return p / (1 + torch.exp(-p)) if name == 'silu' else p


def _slope(p, name):
    if name == 'leaky_relu':
        return torch.where(p >= 0, 1.0, SLOPE)
    s = 1 / (1 + torch.exp(-p))
    return s * (1 + p * (1 - s))


def _grouped(s, t):
    """x-shaped tensor as (N, pixels, groups, channels of a group) or, channels first, (N, groups, channels, pixels);
    the axes of one group, and the shape of per-channel values there."""
    N, C, HW, G = s['N'], s['C'], s['HW'], s['groups']
    if s['last']:
        return t.view(N, HW, G, C // G), (1, 3), (1, 1, G, C // G)
    return t.view(N, G, C // G, HW), (2, 3), (1, G, C // G, 1)


def _plain(s):
    k = s['kind']
    if k == 'keep8':
        q, byte = _codes(s['x'])
        return _kept_values(q, byte, s['n'])
    if k == 'grad8':
        n = s['rows'] * s['K']
        blocks = -(-n // 32)
        x = _kept_values(s['kept'][:32 * blocks].view(torch.int8).view(-1, 32), s['kept'][32 * blocks:], n)
        return x.view(s['rows'], s['K']).t().contiguous() @ s['dy']
    x, axes, per_c = _grouped(s, s['x'])
    gamma, beta = s['gamma'].view(per_c), s['beta'].view(per_c)
    mean = x.mean(axes, keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(axes, keepdim=True) + EPS)
    xh = centred * rstd
    p = xh * gamma + beta
    y = _act(p, s['act']).view(s['x'].shape)
    if k == 'norm':
        return y
    if k == 'train8':     # the backward pass sees what was kept of x
        q, byte = _codes(s['x'].reshape(-1))
        x = _grouped(s, _kept_values(q, byte, s['x'].numel()))[0]
        xh = (x - mean) * rstd
        p = xh * gamma + beta
    dp = _grouped(s, s['dy'])[0]
    if s['act'] != 'none':
        dp = dp * _slope(p, s['act'])
    others = (0, 1) if s['last'] else (0, 3)
    dbeta, dgamma = dp.sum(others).view(-1), (dp * xh).sum(others).view(-1)
    g = dp * gamma
    dx = rstd * (g - g.mean(axes, keepdim=True) - xh * (g * xh).mean(axes, keepdim=True))
    return y, dx.view(s['x'].shape), dgamma, dbeta


def run(s):
    return _own(s) if own else _plain(s)


# ---- from the definitions, in 64 bits ---------------------------------------
def _kept64(x):
    """What the 8-bit copy of x stands for: the step of a block is the smallest power of two 2^e >= 2^-126 for which its
    largest magnitude rounds to 127 or less (2^121 at most)."""
    n = x.numel()
    v = torch.zeros(-(-n // 32) * 32, dtype=torch.float64, device=x.device)
    v[:n] = x
    v = v.view(-1, 32)
    top = v.abs().max(1, keepdim=True).values
    def power(e):         # exactly: pow() is not
        return ((e.long() + 1023) << 52).view(torch.float64)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -140) / 127.5))
    e += ((top / power(e)) >= 127.5).double()        # a largest value of exactly 127.5 steps rounds to 128
    step = power(e.clamp(-126, 121))
    return (torch.round(v / step).clamp(-127, 127) * step).view(-1)[:n]


def exact(case, seed):
    s = _values(case, seed)
    k = case['kind']
    if k == 'keep8':
        return _kept64(s['x'])
    if k == 'grad8':
        return torch.mm(_kept64(s['x'].reshape(-1)).view(case['rows'], case['K']).t(), s['dy'].double())
    N, C, HW, G = case['N'], case['C'], case['HW'], case['groups']
    D = C // G * HW

    def rows(t):          # (N * G, channels of a group, pixels)
        t = t.double()
        t = t.transpose(1, 2) if case['last'] else t
        return t.reshape(N * G, C // G, HW)

    def back(t):
        t = t.view(N, C, HW)
        return t.transpose(1, 2) if case['last'] else t

    def channel(v):
        return v.double().view(1, G, C // G, 1).expand(N, G, C // G, 1).reshape(N * G, C // G, 1)

    def function(p):      # f and f'
        if case['act'] == 'silu':
            sg = torch.sigmoid(p)
            return p * sg, sg + p * sg * (1 - sg)
        if case['act'] == 'leaky_relu':
            return torch.maximum(p, SLOPE * p), None
        return p, torch.ones_like(p)
    x, gamma, beta = rows(s['x']), channel(s['gamma']), channel(s['beta'])
    mean = x.sum((1, 2), keepdim=True) / D
    rstd = ((x - mean).square().sum((1, 2), keepdim=True) / D + EPS).rsqrt()
    y = back(function(gamma * (x - mean) * rstd + beta)[0])
    if k == 'norm':
        return y
    if k == 'train8':
        x = rows(_kept64(s['x'].reshape(-1)).view(s['x'].shape))
    xh = (x - mean) * rstd
    dp = rows(s['dy']) * function(gamma * xh + beta)[1]
    dbeta, dgamma = (t.view(N, C, HW).sum((0, 2)) for t in (dp, dp * xh))
    g = gamma * dp
    dx = rstd * (g - g.sum((1, 2), keepdim=True) / D - xh * ((g * xh).sum((1, 2), keepdim=True) / D))
    return y, back(dx), dgamma, dbeta
