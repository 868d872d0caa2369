"""What the operators on device tensors (recurrence, block_norm, activation8) share: checks of arguments and the way to a kernel's
stream and device."""
import contextlib

import torch

from ac_solver import _acx

DTYPES = {torch.float32: _acx.F32, torch.bfloat16: _acx.BF16, torch.float16: _acx.F16}
_NO_GUARD = contextlib.nullcontext()


def activation(t, name, like=None, shape=None):
    """`t` as a kernel reads it: a tensor of float32 / bfloat16 / float16 whose last axis is contiguous (a copy is made of one whose
    is not, such as the expanded gradient of a sum).  `like`: another activation that it has to match in type and device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} has to be a tensor, not {type(t).__name__}")
    dtype = t.dtype
    if dtype not in DTYPES:
        raise TypeError(f"{name} has to be float32, bfloat16 or float16, not {dtype}")
    if like is not None and (dtype is not like.dtype or t.device != like.device):
        raise ValueError(f"{name} is {dtype} on {t.device}, the other activations are {like.dtype} on {like.device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has the shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t if t.is_contiguous() or t.shape[-1:] == (1,) or t.stride(-1) == 1 else t.contiguous()


def plain(t, name, shape, device, dtype=torch.float32):
    """a contiguous tensor of exactly this type, shape and device (parameters, states, flags)"""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} has to be a tensor, not {type(t).__name__}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} has to be {dtype}, not {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has the shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{name} lives on {t.device}, the activations on {device}")
    return t if t.is_contiguous() else t.contiguous()


def flags(t, name, shape, device):
    """a bool (or uint8) tensor as the kernels read it"""
    if isinstance(t, torch.Tensor) and t.dtype is torch.bool:
        t = t.view(torch.uint8)
    return plain(t, name, shape, device, torch.uint8)


def require_gpu(t):
    """behind the checks of shapes and types, in front of the first allocation"""
    if not t.is_cuda:
        raise ValueError(f"the activations have to live on a GPU, not on {t.device}: there is no CPU path")


def ptr(t):
    return None if t is None else t.data_ptr()


def on_device_of(t):
    """with-block in which kernels go to the device of `t` (a no-op on the current device)"""
    return _NO_GUARD if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def stream_of(t):
    # (torch.cuda.current_stream makes a Stream object first: 2 us of a 10 us call)
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def scratch(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def once(backward):
    """torch.autograd.function.once_differentiable for a backward function that is not being differentiated itself, without its cost: the
    wrapper only matters where autograd records the backward pass (create_graph)."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run
