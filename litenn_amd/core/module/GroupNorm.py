import litenn_amd as nn


class GroupNorm(nn.Module):
    """Group normalisation layer with an activation (see nn.group_norm).

     groups, channels   ints, groups divides channels
     eps(1e-5)
     affine(True)       trainable scale gamma and offset beta per channel
     activation(None)   None | 'leaky_relu' | 'relu' | 'silu';  alpha(0.1) of the leaky ReLU
     channels_last(False)
     keep8(False)       while training (set_training), hold the layer's input in 8 bits for the backward pass
     gamma_initializer  default: nn.initializer.Scalar(1.0)
     beta_initializer   default: nn.initializer.Scalar(0.0)
    """

    def __init__(self, groups, channels, eps=1e-5, affine=True, activation=None, alpha=0.1, channels_last=False, keep8=False,
                 gamma_initializer=None, beta_initializer=None):
        if groups < 1 or channels % groups != 0:
            raise ValueError(f'groups must divide the channels: {groups} and {channels}')
        self.groups, self.channels, self.eps, self.affine = groups, channels, eps, affine
        self.activation, self.alpha, self.channels_last, self.keep8 = activation, alpha, channels_last, keep8
        self.gamma = self.beta = None
        if affine:
            self.gamma = nn.Tensor((channels,), init=gamma_initializer or nn.initializer.Scalar(1.0))
            self.beta = nn.Tensor((channels,), init=beta_initializer or nn.initializer.Scalar(0.0))
        super().__init__(saveables=['gamma', 'beta'])

    def forward(self, x, **kwargs):
        return nn.group_norm(x, self.groups, self.gamma, self.beta, self.eps, self.activation, self.alpha, self.channels_last,
                             keep8=self.keep8 and self.is_training())

    def __str__(self): return f'{self.__class__.__name__} : groups:{self.groups} channels:{self.channels} '
    __repr__ = __str__
