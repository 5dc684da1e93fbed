"""Per-pixel decoding of rendered feature images on the HIP library.

``rasterize`` renders learned features as channel-last images (..., H, W, D);
a decoder of per-pixel products and group norms takes them into the space in
which they are trained.  Its operators: ``linear`` (product, bias, activation,
residual), ``group_norm`` (with an activation) and ``quantize_activations``,
the 8-bit form in which either may keep its input for the backward pass.
``FeatureDecoder`` is a small network of them.
"""

from .activations import QuantizedActivations, quantize_activations
from .decoder import FeatureDecoder
from .linear import linear
from .norm import group_norm

__all__ = ["linear", "group_norm", "quantize_activations", "QuantizedActivations", "FeatureDecoder"]
