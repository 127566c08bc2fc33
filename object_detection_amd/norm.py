"""Group norm fused with the activation that follows it, on channels-last maps.

The head towers of the reference's models are [conv, GroupNorm(32), ReLU] blocks (``partial(nn.GroupNorm, 32)`` at
``object_detection/retinanet/retinanet_model.py:47-52``; torchvision's FCOS head builds the same).  Convolutions run in
channels-last memory on this hardware and hand on channels-last maps; ``GroupNormAct`` keeps them so, where
``nn.GroupNorm`` answers with an NCHW tensor that the next convolution has to lay out again.  Forward and backward are
HIP kernels (``od_group_norm_act_*``); there is no CPU path.
"""
from __future__ import annotations

from typing import Optional

from torch import Tensor, nn

from . import _C, kernels

_ACTIVATIONS = {"none": _C.ACT_NONE, "relu": _C.ACT_RELU, "silu": _C.ACT_SILU}


def group_norm_act(x: Tensor, num_groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                   eps: float = 1e-5, activation: str = "relu") -> Tensor:
    """``act(group_norm(x, num_groups, weight, bias, eps))`` of a map [B, C, H, W] on the GPU (fp32 / fp16 / bf16).

    The result has x's type and channels-last memory; x in another memory order is copied once.  ``activation``: "none",
    "relu" or "silu".  weight / bias [C] share one type, which may differ from x's (fp32 parameters of a tower that runs
    under autocast).  Statistics are merged and kept in 64 bits, everything else is fp32 for every type; the result is
    rounded once.  Differentiable once in x, weight and bias.  Limits: 2048 channels, 65535 images."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {sorted(_ACTIVATIONS)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return kernels.group_norm_act(x, num_groups, weight, bias, eps, _ACTIVATIONS[activation])


class GroupNormAct(nn.GroupNorm):
    """``nn.GroupNorm`` with the activation behind it in the same kernel.  Same parameters and state-dict keys;
    ``partial(GroupNormAct, 32)`` is a ``norm_layer`` for the heads and ``get_model``, whose towers then leave the place of
    their ReLU to an ``nn.Identity``, so that checkpoints of either form load into the other."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: str = "relu", device=None, dtype=None):
        if activation not in _ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}: one of {sorted(_ACTIVATIONS)}")
        super().__init__(num_groups, num_channels, eps, affine, device=device, dtype=dtype)
        self.activation = activation

    def forward(self, x: Tensor) -> Tensor:
        return group_norm_act(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self) -> str:
        return super().extra_repr() + f", activation={self.activation}"


def activates(norm: nn.Module) -> bool:
    """Whether a norm layer already applies the activation of its block."""
    return isinstance(norm, GroupNormAct) and norm.activation != "none"
