"""Argument checks and layouts that the decoder's operators share."""

import torch
from torch import Tensor
from torch.autograd import forward_ad

from ..runtime import abi, native

DTYPES = {torch.float32: abi.DTYPE_F32, torch.bfloat16: abi.DTYPE_BF16, torch.float16: abi.DTYPE_F16}
ACTIVATIONS = {"none": abi.ACT_NONE, "relu": abi.ACT_RELU, "silu": abi.ACT_SILU, "gelu": abi.ACT_GELU}
CHECKPOINTS = (None, "int8")


def check_input(name: str, x: Tensor, least_dims: int) -> None:
    if not (isinstance(x, Tensor) and x.is_cuda and x.dtype in DTYPES):
        raise ValueError(f"{name} must be a CUDA float32, bfloat16 or float16 tensor")
    if x.ndim < least_dims or x.shape[-1] < 1:
        raise ValueError(f"{name} must have at least {least_dims} dimensions and one channel")
    if x.shape[-1] > abi.MAX_CHANNELS:
        raise ValueError(f"{name} has {x.shape[-1]} channels, more than {abi.MAX_CHANNELS}")
    if x.numel() // x.shape[-1] > abi.MAX_ROWS:
        raise ValueError(f"{name} has more than {abi.MAX_ROWS} pixels")


def check_like(name: str, tensor: Tensor | None, x: Tensor, shape: tuple[int, ...]) -> None:
    """ValueError unless `tensor` is None or of x's dtype and device and of `shape`."""
    if tensor is None:
        return
    if not (isinstance(tensor, Tensor) and tensor.dtype == x.dtype and tensor.device == x.device):
        raise ValueError(f"{name} must be {x.dtype} on {x.device}")
    if tuple(tensor.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(tensor.shape)}")


def activation_code(activation: str) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def check_checkpoint(checkpoint: str | None) -> None:
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"checkpoint must be one of {CHECKPOINTS}, got {checkpoint!r}")


def rows_of(x: Tensor) -> tuple[Tensor, int]:
    """(tensor, row stride): x as rows of contiguous channels a uniform stride
    apart, copied only where it is not laid out like that."""
    channels = x.shape[-1]
    if x.is_contiguous():
        return x, channels
    if channels == 1 or x.stride(-1) == 1:
        # Leading dimensions of one element have any stride.
        dims = [(n, s) for n, s in zip(x.shape[:-1], x.stride()[:-1]) if n != 1]
        if not dims:
            return x, channels
        if dims[-1][1] >= channels and all(a[1] == b[0] * b[1] for a, b in zip(dims, dims[1:])):
            return x, dims[-1][1]
    return x.contiguous(), channels


def scratch(nbytes: int, device: torch.device) -> Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def recorded(*tensors: Tensor | None) -> bool:
    """Whether autograd has to see a call on these tensors.  One that it need
    not see runs without a node (10 us rather than 15 of host time); within
    forward-mode differentiation all are shown, and refused by the node, and a
    trace keeps the node where it would keep nothing of a launch."""
    if getattr(forward_ad, "_current_level", 0) >= 0 or torch.jit.is_tracing():
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def check_untraced(name: str) -> None:
    """RuntimeError while torch.jit.trace records: it would keep an operator
    without a node as an uninitialised tensor."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{name} cannot be traced")


def launch(name: str, args, device: torch.device, *rest) -> None:
    """native.call on the current stream of `device`."""
    if device.index is None or device.index == torch.cuda.current_device():
        native.call(name, args, *rest, native.stream(device))
    else:
        with torch.cuda.device(device):
            native.call(name, args, *rest, native.stream(device))
