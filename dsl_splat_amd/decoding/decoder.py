"""A per-pixel network over rendered feature images."""

import torch
from torch import Tensor, nn

from .linear import linear
from .norm import group_norm


class FeatureDecoder(nn.Module):
    """Rendered features (..., H, W, in_channels) to (..., H, W, out_channels):

        h = act(x W_in^T + b_in)
        h = h + (act(group_norm(h)) W_i^T + b_i)      for every block
        y = h W_out^T + b_out

    with checkpoint="int8" every operator keeps its input in 8 bits for the
    backward pass.  The input is cast to the parameters' dtype.

        res = gs3d.rasterize(..., features=features)
        loss = (decoder(res.features) - teacher).square().mean()
    """

    def __init__(self, in_channels: int, hidden: int, out_channels: int, *, blocks: int = 1, groups: int = 8,
                 activation: str = "silu", checkpoint: str | None = None, device=None, dtype=torch.float32):
        super().__init__()
        if hidden % groups:
            raise ValueError(f"groups must divide the {hidden} hidden channels, got {groups}")
        self.groups, self.activation, self.checkpoint = groups, activation, checkpoint
        widths = [(in_channels, hidden)] + [(hidden, hidden)] * blocks + [(hidden, out_channels)]
        make = dict(device=device, dtype=dtype)
        self.weights = nn.ParameterList(torch.randn((n, k), **make) * k ** -0.5 for k, n in widths)
        self.biases = nn.ParameterList(torch.zeros((n,), **make) for _, n in widths)
        self.scales = nn.ParameterList(torch.ones((hidden,), **make) for _ in range(blocks))
        self.shifts = nn.ParameterList(torch.zeros((hidden,), **make) for _ in range(blocks))

    def forward(self, features: Tensor) -> Tensor:
        keep = dict(checkpoint=self.checkpoint)
        h = linear(features.to(self.weights[0].dtype), self.weights[0], self.biases[0], activation=self.activation,
                   **keep)
        for i, (scale, shift) in enumerate(zip(self.scales, self.shifts), start=1):
            a = group_norm(h, self.groups, scale, shift, activation=self.activation, **keep)
            h = linear(a, self.weights[i], self.biases[i], residual=h, **keep)
        return linear(h, self.weights[-1], self.biases[-1], **keep)
