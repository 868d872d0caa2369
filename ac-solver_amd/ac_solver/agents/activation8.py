"""Activations kept in 8 bits for the backward pass, and the weight gradient that reads them as they are: `acx_act8_pack` / `_unpack` /
`_weight_grad` (csrc/acx_act8.hip).  Opt-in (`--checkpoint-8bit` of ac_solver.agents.ppo); the reference keeps float32 activations
(ac_solver/agents/ppo_agent.py:11-109, agents/training.py:273-330)."""
import threading

import torch
from torch.nn import functional as F

from ac_solver import _acx
from ac_solver.agents import _tensors as T

BLOCK = 32


def _checkpoint(q, exponent):
    q = T.plain(q, "q", q.shape if isinstance(q, torch.Tensor) else (), q.device if isinstance(q, torch.Tensor) else None, torch.int8)
    if q.dim() < 1:
        raise ValueError("q has to have a feature axis")
    return q, T.plain(exponent, "exponent", q.shape[:-1] + (-(-q.shape[-1] // BLOCK),), q.device, torch.uint8)


def pack8(x):
    """x [..., width] (float32, bfloat16 or float16) -> (q [..., width] int8, exponent [..., ceil(width / 32)] uint8): the value kept for x
    is q * 2^(exponent - 127), with one exponent for 32 neighbouring features -- the smallest for which the largest of them rounds to at
    most 127, so the error is at most 2^-7 of that largest one.  A block that holds an infinity or a NaN is marked (exponent 255) and
    restores to NaN."""
    x = T.activation(x, "x")
    if x.dim() < 1:
        raise ValueError("x has to have a feature axis")
    width = x.shape[-1]
    T.require_gpu(x)
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    exponent = torch.empty(x.shape[:-1] + (-(-width // BLOCK),), dtype=torch.uint8, device=x.device)
    if x.numel():
        x2 = x.reshape(-1, width)
        with T.on_device_of(x):
            _acx.check(_acx.lib.acx_act8_pack(x2.data_ptr(), x2.stride(0), T.DTYPES[x.dtype], x2.shape[0], width, q.data_ptr(), exponent.data_ptr(), T.stream_of(x)), "acx_act8_pack")
    return q, exponent


def unpack8(q, exponent, dtype=torch.float32):
    """the values that a checkpoint of pack8 stands for, rounded to `dtype` (exact in float32 and bfloat16)"""
    if dtype not in T.DTYPES:
        raise TypeError(f"dtype has to be float32, bfloat16 or float16, not {dtype}")
    q, exponent = _checkpoint(q, exponent)
    T.require_gpu(q)
    x = torch.empty(q.shape, dtype=dtype, device=q.device)
    if q.numel():
        with T.on_device_of(q):
            _acx.check(_acx.lib.acx_act8_unpack(q.data_ptr(), exponent.data_ptr(), q.numel() // q.shape[-1], q.shape[-1], x.data_ptr(), T.DTYPES[dtype], T.stream_of(q)),
                       "acx_act8_unpack")
    return x


def weight_grad8(d_out, q, exponent):
    """The gradients of weight and bias of a linear layer whose input was kept by pack8: d_out [..., outputs] (float32, bfloat16 or float16),
    q [..., inputs] -> (d_out^T x [outputs, inputs], sum of d_out [outputs]), both float32, x the values the checkpoint stands for; float32
    accuracy for every type of d_out."""
    d_out = T.activation(d_out, "d_out")
    q, exponent = _checkpoint(q, exponent)
    if d_out.dim() < 1 or d_out.shape[:-1] != q.shape[:-1] or d_out.device != q.device:
        raise ValueError(f"d_out {tuple(d_out.shape)} on {d_out.device} and q {tuple(q.shape)} on {q.device} do not have their rows in common")
    outputs, inputs = d_out.shape[-1], q.shape[-1]
    if outputs > 65536 or inputs > 65536:
        raise ValueError("up to 65536 outputs and inputs")
    T.require_gpu(d_out)
    dev = d_out.device
    rows = q.numel() // inputs if inputs else 0
    if not rows or not outputs:
        return torch.zeros((outputs, inputs), device=dev), d_out.reshape(-1, outputs).float().sum(0) if outputs else torch.zeros(0, device=dev)
    g = d_out.reshape(-1, outputs)
    if rows > 1 and not outputs <= g.stride(0) < 1 << 24:  # (the expanded gradient of a sum over the rows, say)
        g = g.contiguous()
    stride = g.stride(0) if rows > 1 else outputs
    dw = torch.empty((outputs, inputs), dtype=torch.float32, device=dev)
    db = torch.empty(outputs, dtype=torch.float32, device=dev)
    work = T.scratch(_acx.lib.acx_act8_workspace_bytes(rows, outputs, inputs), dev)
    with T.on_device_of(d_out):
        _acx.check(_acx.lib.acx_act8_weight_grad(g.data_ptr(), stride, T.DTYPES[d_out.dtype], q.data_ptr(), exponent.data_ptr(), rows, outputs, inputs, dw.data_ptr(),
                                                 db.data_ptr(), T.ptr(work), 0 if work is None else work.numel(), T.stream_of(d_out)), "acx_act8_weight_grad")
    return dw, db


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        out = F.linear(x, weight.to(x.dtype), None if bias is None else bias.to(x.dtype))
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(*pack8(x), weight)
        return out

    @staticmethod
    @T.once
    def backward(ctx, d_out):
        q, exponent, weight = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad
        dx = d_out @ weight.to(d_out.dtype) if need_x else None
        dw, db = weight_grad8(d_out, q, exponent) if need_w or need_b else (None, None)
        return dx, dw if need_w else None, db if need_b else None


def linear8(x, weight, bias=None):
    """torch.nn.functional.linear with float32 parameters [outputs, inputs], [outputs], computed in the type of x; what it keeps for the
    backward pass is x in 8 bits (pack8), and the gradient of the weight is taken from that (weight_grad8).  The gradient of x is the
    library's and knows nothing of the 8 bits."""
    if not isinstance(weight, torch.Tensor) or weight.dtype != torch.float32 or weight.dim() != 2:
        raise TypeError("weight has to be a float32 matrix")
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.dtype != torch.float32 or bias.shape != weight.shape[:1]):
        raise TypeError("bias has to be a float32 vector, one value for each output")
    x = T.activation(x, "x")
    if x.shape[-1:] != weight.shape[1:]:
        raise ValueError(f"x has the shape {tuple(x.shape)}, the weight {tuple(weight.shape)}")
    T.require_gpu(x)
    return _Linear8.apply(x, weight, bias)


class _Packed:
    """a tensor that autograd saved, in 8 bits; knows the type to restore"""

    __slots__ = ("q", "exponent", "dtype")

    def __init__(self, t):
        self.q, self.exponent = pack8(t)
        self.dtype = t.dtype


MIN_VALUES = 1 << 12
_inside = threading.local()


def packing():
    """whether this thread is inside a `checkpoint8` block (for functions that keep tensors which autograd does not know)"""
    return getattr(_inside, "depth", 0) > 0


class checkpoint8(torch.autograd.graph.saved_tensors_hooks):
    """`with checkpoint8(): ...` -- what autograd keeps of the activations computed inside the block is kept in 8 bits (pack8) and restored
    in the backward pass: a quarter (float32) or half (16 bits) of the memory; the gradients are those of the restored values (row
    statistics and states that an operator kept beside them stay what they were).  Kept as they are: leaves (parameters, inputs),
    vectors, tensors of fewer than 4096 values, whole numbers, tensors on the CPU."""

    def __init__(self):
        super().__init__(self._keep, self._restore)

    def __enter__(self):
        _inside.depth = getattr(_inside, "depth", 0) + 1
        return super().__enter__()

    def __exit__(self, *exc):
        _inside.depth -= 1
        return super().__exit__(*exc)

    @staticmethod
    def _keep(t):
        if t.dtype not in T.DTYPES or not t.is_cuda or t.dim() < 2 or t.numel() < MIN_VALUES or t.grad_fn is None:
            return t
        return _Packed(t)

    @staticmethod
    def _restore(kept):
        return unpack8(kept.q, kept.exponent, kept.dtype) if isinstance(kept, _Packed) else kept
