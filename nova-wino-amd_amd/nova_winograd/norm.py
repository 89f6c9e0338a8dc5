"""Group norm with SiLU on the gfx950 library: ``nova_group_norm`` and the
module ``NovaGroupNorm``, forward and backward, NCHW and channels-last.

No counterpart in the reference, whose package holds the convolution alone: in
a UNet this is what stands between two of its convolutions, and it keeps the
activations in the layout that the convolutions run in.
"""


import torch.nn as nn

from nova_winograd.ops import native

_ACTIVATIONS = {None: False, "silu": True}


def _silu(name, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{name}: activation {activation!r}; None and 'silu' are supported")
    return _ACTIVATIONS[activation]


def nova_group_norm(input, num_groups, weight=None, bias=None, eps=1e-5, activation=None):
    """Group norm over ``num_groups`` groups of channels, followed by the
    activation in the same pass.

    Args:
        input:      [B, C, ...] float16, bfloat16 or float32 tensor on the GPU,
                    contiguous or channels-last (4-d and 5-d); other strides
                    are copied first.
        num_groups: divides C.
        weight:     optional [C] tensor, float16, bfloat16 or float32.
        bias:       optional [C] tensor (converted to ``weight``'s type where
                    that differs).
        eps:        added to the variance.
        activation: None or "silu".

    Returns a tensor of the input's shape, type and layout. Statistics are
    float32; every value is rounded once. Differentiable (once, in reverse
    mode) with respect to input, weight and bias. Runs on PyTorch's current
    stream.
    """
    silu = _silu("nova_group_norm", activation)
    if not isinstance(num_groups, int):
        raise ValueError(f"nova_group_norm: num_groups ({num_groups!r}) is not an integer")
    return native().group_norm(input, num_groups, weight, bias, eps, silu)


class NovaGroupNorm(nn.GroupNorm):
    """``nn.GroupNorm`` (same parameters and state dict) through
    ``nova_group_norm``, with the activation behind it taken in."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation=None,
                 device=None, dtype=None):
        _silu("NovaGroupNorm", activation)
        super().__init__(num_groups, num_channels, eps=eps, affine=affine, device=device,
                         dtype=dtype)
        self.activation = activation

    @classmethod
    def from_group_norm(cls, norm, activation=None):
        """A module with copies of ``nn.GroupNorm`` ``norm``'s parameters."""
        p = norm.weight
        mod = cls(norm.num_groups, norm.num_channels, eps=norm.eps, affine=norm.affine,
                  activation=activation, device=None if p is None else p.device,
                  dtype=None if p is None else p.dtype)
        mod.load_state_dict(norm.state_dict())
        return mod

    def forward(self, input):
        return nova_group_norm(input, self.num_groups, self.weight, self.bias, self.eps,
                               self.activation)

    def extra_repr(self):
        return f"{super().extra_repr()}, activation={self.activation}"
