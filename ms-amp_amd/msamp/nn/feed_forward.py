"""FeedForward: the two or three linear layers of a transformer's feed-forward block, which run as fused FP8 products once
they are FP8Linear layers (not in the reference, which has no blocks)."""

import torch
import torch.nn.functional as F

from msamp.nn.linear import FP8Linear
from msamp.operators.activation import Activation

_TORCH = {
    'relu': F.relu,
    'gelu': F.gelu,
    'gelu_tanh': lambda x: F.gelu(x, approximate='tanh'),
    'silu': F.silu,
}


class FeedForward(torch.nn.Module):
    """down(act(up(x))) or, with a gate layer, down(act(gate(x)) * up(x)); `residual`, if given to the call, is added to it.

    Built from linear layers, before or after msamp.initialize has replaced them.  FP8Linear layers take activation, gate and
    residual into their products and keep what the activation's backward pass needs in 8 bits: beside the codes of the products'
    inputs one byte and 1/32 for every hidden value, two with a gate, where element-wise operators keep 4 to 8; all of it is freed
    behind the backward pass.  For training and for prompts: of up to 64 tokens the plain layers take less (linear_fused)."""

    def __init__(self, up, down, gate=None, activation='gelu'):
        super().__init__()
        if activation not in Activation.NAMES:
            raise ValueError(f'unknown activation {activation!r}: one of {", ".join(Activation.NAMES)}')
        self.up, self.down, self.gate = up, down, gate
        self.activation = activation

    def forward(self, x, residual=None):
        first = self.up if self.gate is None else self.gate
        beside = None if self.gate is None else self.up(x)
        if isinstance(first, FP8Linear):
            hidden = first(x, activation=self.activation, gate=beside)
        else:
            hidden = _TORCH[self.activation](first(x))
            hidden = hidden if beside is None else hidden * beside
        if residual is None:
            return self.down(hidden)
        return self.down(hidden, residual=residual) if isinstance(self.down, FP8Linear) else self.down(hidden) + residual

    def extra_repr(self):
        return f'activation={self.activation}'
