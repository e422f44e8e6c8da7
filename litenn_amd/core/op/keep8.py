import litenn_amd as nn


def keep8(t):
    """Hold tensor t in 8 bits from here on: what a forward pass leaves for the backward pass takes a quarter of its
    memory.  (A dense layer's weight gradient then needs scratch, one for all layers: 2 bytes per element of its input and
    6 per element of its output gradient, at most about a gigabyte.)

    The fp32 storage goes back to the pool; every 32 elements that follow each other in memory share a power of two and
    are rounded to 7 bits and sign below it (off by at most 1 / 127 of the largest of the 32).  Call it when the forward
    pass has read t for the last time:

        h = conv1(x)
        y = nn.group_norm(h, 8, gamma, beta, activation='silu')
        nn.keep8(h)                      # or group_norm(..., keep8=True): written while the norm reads h
        z = dense(y.reshape(...)); nn.keep8(y)

    The gradient functions of group_norm and of a matmul's second operand (a dense layer's weight) read the copy as it
    is; every other reader of t, forward or backward, gets the rounded values decoded into fp32, which backward() lets go
    again as soon as the tensor's gradient functions have run.  A value below half a step reads back as 0, also for a
    (leaky) ReLU whose gradient takes the sign from t.  Writing to t (set, fill, output_t=) ends the 8-bit state.
    Returns t."""
    check_keep8(t)
    for buf in t._get_buffers():
        buf.keep8()
    return t


def check_keep8(t):
    """ValueError for tensors that are not to be held in 8 bits."""
    if not isinstance(t, nn.Tensor):
        raise ValueError(f'keep8 expects a Tensor, not {t.__class__}')
    if t._is_grad():
        raise ValueError('keep8: gradients stay in fp32')
    if t._is_trainable() or t._get_top_reference_source()._parent_module_w is not None:
        raise ValueError(f'keep8: {t.get_name()} is a parameter, parameters stay in fp32')
