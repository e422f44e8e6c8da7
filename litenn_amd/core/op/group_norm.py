import litenn_amd as nn
import litenn_amd.core as nc
from ..backward import after_gradfns_of_tensor, current_sweep, gradient_wanted
from ..hip import api, hold8, kept8, launch, new_kept8

_ACTS = {None: api.ACT_NONE, 'leaky_relu': api.ACT_LEAKY_RELU, 'relu': api.ACT_LEAKY_RELU, 'silu': api.ACT_SILU}


def group_norm(input_t, groups, gamma_t=None, beta_t=None, eps=1e-5, activation=None, alpha=0.1, channels_last=False,
               keep8=False):
    """Group normalisation and the activation behind it, in one operator.

     input_t        (batch, channels, ...), or (batch, ..., channels) with channels_last; (rows, channels), the output
                    of a dense layer, is either
     groups         int that divides channels.  The elements of one image in channels / groups neighbouring channels
                    are normalised together: (x - mean) / sqrt(var + eps)
     gamma_t        (channels,) scale, default 1
     beta_t         (channels,) offset, default 0
     activation     None | 'leaky_relu' (x >= 0 ? x : alpha*x) | 'relu' | 'silu' (x / (1 + exp(-x)))
     keep8          hold input_t in 8 bits from here on, as nn.keep8(input_t) does, the copy written in the same pass.
                    input_t must not be a parameter or gradient.
    Tensors of less than 2 GiB, at most 4194304 channels.

    Gradients of input, gamma and beta, each accumulated, are formed together in one pass over input and output
    gradient; the activation's slope is formed again from the input.
    """
    if activation not in _ACTS:
        raise ValueError(f'unknown activation {activation!r}: {", ".join(repr(a) for a in _ACTS)} are known')
    if groups != int(groups):
        raise ValueError(f'groups must be a whole number: {groups}')
    op = nc.Cacheton.get(_GroupNormOp, input_t.shape, int(groups), bool(channels_last), float(eps), activation,
                         float(alpha) if activation == 'leaky_relu' else 0.0)
    for name, t in (('gamma', gamma_t), ('beta', beta_t)):
        if t is not None and tuple(t.shape) != (op.channels,):
            raise ValueError(f'{name} shape {tuple(t.shape)} does not match {op.channels} channels')
    if keep8:
        nc.op.check_keep8(input_t)
    output_t = nn.Tensor(input_t.shape)
    output_t._set_op_name('group_norm')
    mean_t, rstd_t = nn.Tensor(op.rows_shape), nn.Tensor(op.rows_shape)
    grad = _GroupNormGrad(op, input_t, gamma_t, beta_t, mean_t, rstd_t)
    for which, t in enumerate((input_t, gamma_t, beta_t)):
        if t is not None:
            output_t._assign_gradfn(t, lambda O_t, dO_t, which=which: grad(which, O_t, dO_t))
    x8 = new_kept8(input_t) if keep8 else None
    launch(lambda dev, *p: api.group_norm_fwd(dev, op.desc, *p), (input_t, 'r'), _read(gamma_t), _read(beta_t), (output_t, 'w'),
           (mean_t, 'w'), (rstd_t, 'w'), None if x8 is None else (x8, 'w'))
    if keep8:
        hold8(input_t, x8)
    return output_t


def _read(t):
    return None if t is None else (t, 'r')


class _GroupNormGrad:
    """Backward of one group_norm result: its gradient functions share one pass, run by whichever backward() calls
    first."""

    def __init__(self, op, input_t, gamma_t, beta_t, mean_t, rstd_t):
        self.op, self.inputs, self.stats = op, (input_t, gamma_t, beta_t), (mean_t, rstd_t)
        self.done = None      # (backward sweep, dO tensor) that the gradients were formed for

    def _drop(self):
        self.done = None

    def __call__(self, which, O_t, dO_t):
        sweep = current_sweep()
        if sweep is None:      # called outside backward(): this gradient alone
            self._run([which], dO_t)
            return
        if self.done is not None and self.done[0] == sweep and self.done[1] is dO_t:
            return
        wanted = [i for i, t in enumerate(self.inputs) if t is not None and gradient_wanted(O_t, t)]
        if len({id(self.inputs[i]._get_top_reference_source()) for i in wanted}) < len(wanted):
            for i in wanted:   # one tensor in two places: its gradient is added to twice, one launch behind the other
                self._run([i], dO_t)
        else:
            self._run(wanted, dO_t)
        self.done = (sweep, dO_t)
        after_gradfns_of_tensor(self._drop)

    def _run(self, wanted, dO_t):
        input_t, gamma_t, beta_t = self.inputs
        outs, betas = [None] * 3, [0] * 3
        for i in wanted:
            outs[i], betas[i] = nc.op.accumulate_target(self.inputs[i].get_grad())
        x8 = kept8(input_t)
        launch(lambda dev, *p: api.group_norm_bwd(dev, self.op.desc, *p, *betas), None if x8 is not None else (input_t, 'r'), _read(x8),
               _read(gamma_t), _read(beta_t), (self.stats[0], 'r'), (self.stats[1], 'r'), (dO_t, 'r'), *outs)


class _GroupNormOp:
    """Shape plan of one group norm, memoised by Cacheton."""

    def __init__(self, shape, groups, channels_last, eps, activation, alpha):
        if shape.rank < 2:
            raise ValueError('group_norm expects (batch, channels, ...) or, channels last, (batch, ..., channels).')
        C = shape[-1] if channels_last else shape[1]
        if groups < 1 or C % groups != 0:
            raise ValueError(f'groups must divide the channels: {groups} and {C}')
        if not eps > 0:
            raise ValueError('eps must be > 0')
        N = shape[0]
        self.channels = C
        self.rows_shape = nc.TensorShape((N, groups))
        self.desc = api.group_norm_desc(N, C, shape.size // (N * C), groups, channels_last, _ACTS[activation], alpha, eps)
