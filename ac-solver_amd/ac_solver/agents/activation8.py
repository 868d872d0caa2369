"""Activations kept in 8 bits for the backward pass, and the weight gradient that reads them as they are: `acx_act8_pack` / `_unpack` /
`_weight_grad` (csrc/acx_act8.hip).  Opt-in (`--checkpoint-8bit` of ac_solver.agents.ppo); the reference keeps float32 activations
(ac_solver/agents/ppo_agent.py:11-109, agents/training.py:273-330)."""
import re
import threading

import torch
from torch.nn import functional as F

from ac_solver.agents._ops import DTYPES, ops


def pack8(x):
    """x [..., width] (float32, bfloat16 or float16) -> (q [..., width] int8, exponent [..., ceil(width / 32)] uint8): the value kept for x
    is q * 2^(exponent - 127), with one exponent for 32 neighbouring features -- the smallest for which the largest of them rounds to at
    most 127, so the error is at most 1/127 of that largest one, or 2^-127 (rows of up to 2^20 features).  A block that holds an infinity or a NaN is marked (exponent
    255) and restores to NaN; finite values restore to finite ones (see unpack8)."""
    return ops.pack8(x)


def unpack8(q, exponent, dtype=torch.float32):
    """the values that a checkpoint of pack8 stands for, rounded to `dtype` (exact in float32 and bfloat16); what lies above the largest finite value of `dtype`
    (float16's 65504 is kept as 64 * 2^10, float32's largest as 64 * 2^122) becomes that largest value"""
    if not isinstance(dtype, torch.dtype):
        raise TypeError(f"dtype has to be a torch type, not {type(dtype).__name__}")
    return ops.unpack8(q, exponent, dtype)


def weight_grad8(d_out, q, exponent):
    """The gradients of weight and bias of a linear layer whose input was kept by pack8: d_out [..., outputs] (float32, bfloat16 or float16),
    q [..., inputs] -> (d_out^T x [outputs, inputs], sum of d_out [outputs]), both float32, x the values the checkpoint stands for (unpack8 in
    bfloat16); float32 accuracy for every type of d_out.  Up to 65536 outputs and inputs, 2^29 weights."""
    return ops.weight_grad8(d_out, q, exponent)


MAX_SIDE, MAX_WEIGHTS = 1 << 16, 1 << 29  # of weight_grad8


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        out = F.linear(x, weight.to(x.dtype), None if bias is None else bias.to(x.dtype))
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(*pack8(x), weight)
        return out

    @staticmethod
    def backward(ctx, d_out):
        q, exponent, weight = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad
        with torch.no_grad():
            dx = d_out @ weight.to(d_out.dtype) if need_x else None
            dw, db = weight_grad8(d_out, q, exponent) if need_w or need_b else (None, None)
        grads = dx, dw if need_w else None, db if need_b else None
        return ops.once(grads, d_out) if torch.is_grad_enabled() else grads


def linear8(x, weight, bias=None):
    """torch.nn.functional.linear with float32 parameters [outputs, inputs], [outputs], computed in the type of x; what it keeps for the
    backward pass is x in 8 bits (pack8), and the gradient of the weight is taken from that (weight_grad8, whose sizes are the limit of a
    layer that wants one).  The gradient of x is the library's and knows nothing of the 8 bits.  Differentiable once."""
    if not isinstance(weight, torch.Tensor) or weight.dtype != torch.float32 or weight.dim() != 2:
        raise TypeError("weight has to be a float32 matrix")
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.dtype != torch.float32 or bias.shape != weight.shape[:1]):
        raise TypeError("bias has to be a float32 vector, one value for each output")
    if not isinstance(x, torch.Tensor) or x.dtype not in DTYPES:
        raise TypeError("x has to be a float32, bfloat16 or float16 tensor")
    if x.shape[-1:] != weight.shape[1:]:
        raise ValueError(f"x has the shape {tuple(x.shape)}, the weight {tuple(weight.shape)}")
    outputs, inputs = weight.shape
    if torch.is_grad_enabled() and (weight.requires_grad or (bias is not None and bias.requires_grad)) and (outputs > MAX_SIDE or inputs > MAX_SIDE or outputs * inputs > MAX_WEIGHTS):
        raise ValueError(f"the gradient of a layer of up to {MAX_SIDE} outputs and inputs and {MAX_WEIGHTS} weights is handled, not of {outputs} x {inputs}")
    if not x.is_cuda:
        raise ValueError(f"the activations have to live on a GPU, not on {x.device}: there is no CPU path")
    return _Linear8.apply(x, weight, bias)


class _Packed:
    """a tensor that autograd saved, in 8 bits; knows the type to restore"""

    __slots__ = ("q", "exponent", "dtype")

    def __init__(self, t):
        self.q, self.exponent = pack8(t)
        self.dtype = t.dtype

    def restore(self):
        return unpack8(self.q, self.exponent, self.dtype)


class _Kept:
    """a tensor that autograd saved, as it is.  (Detached: autograd hangs it back into its graph; the tensor itself, if its own node keeps it, would hold that
    node, and the graph behind it, for good.)  Autograd leaves it to the hooks to notice that it has been changed in place since."""

    __slots__ = ("tensor", "version")

    def __init__(self, t):
        self.tensor = t.detach()
        self.version = None if t.is_inference() else t._version

    def restore(self):
        t = self.tensor
        if self.version is not None and t._version != self.version:
            raise RuntimeError(f"one of the variables needed for gradient computation has been modified by an inplace operation: {tuple(t.shape)} of {t.dtype} is at version "
                               f"{t._version}, expected version {self.version}")
        return t


MIN_VALUES = 1 << 12  # a tensor worth a launch
MAX_WIDTH = 1 << 20  # of pack8
_inside = threading.local()


def packing():
    """whether this thread is inside a `checkpoint8` block (for functions that keep tensors which autograd does not know)"""
    return getattr(_inside, "depth", 0) > 0


# nodes of autograd that hand a tensor on with the same values, up to a rounding to another type (torch's own have a number behind their names)
_SAME_VALUES = re.compile("(Alias|AsStrided|Clone|Diagonal|Expand|Movedim|Permute|ReshapeAlias|Select|Slice|Split|SplitWithSizes|Squeeze|T|ToCopy|Transpose|Unbind|Unfold|UnsafeSplit|UnsafeView|"
                          "Unsqueeze|View)Backward[0-9]+")


def _is_leaf(t):
    """whether t is a leaf (a parameter, an input), a view of one, or a copy of one in another type or layout: torch's linear layer keeps the transpose of
    its weight, in bfloat16 that of a copy which autocast made.  (A view that a function made without recording it has a base without a
    gradient of its own: the function's result, not a leaf.)"""
    if t.grad_fn is None or (t._base is not None and t._base.is_leaf and t._base.requires_grad):
        return True
    node = t.grad_fn
    while _SAME_VALUES.fullmatch(node.name()):
        node = node.next_functions[0][0]
        if node is None:
            return True
    return node.name().endswith("AccumulateGrad")


class checkpoint8(torch.autograd.graph.saved_tensors_hooks):
    """`with checkpoint8(): ...` -- what autograd keeps of the activations computed inside the block is kept in 8 bits (pack8) and restored
    in the backward pass: a quarter (float32) or half (16 bits) of the memory; the gradients are those of the restored values (row
    statistics and states that an operator kept beside them stay what they were).  Kept as they are: leaves (parameters, inputs), their
    views and their copies in other types, vectors, tensors with one value a row (row statistics), of fewer than 4096 values or with rows of more
    than 2^20, whole numbers, tensors on the CPU."""

    def __init__(self):
        super().__init__(self._keep, self._restore)

    def __enter__(self):
        super().__enter__()
        _inside.depth = getattr(_inside, "depth", 0) + 1

    def __exit__(self, *exc):
        _inside.depth -= 1
        return super().__exit__(*exc)

    @staticmethod
    def _keep(t):
        if t.dtype not in DTYPES or not t.is_cuda or t.dim() < 2 or t.numel() < MIN_VALUES or not 1 < t.shape[-1] <= MAX_WIDTH or _is_leaf(t):
            return _Kept(t)
        return _Packed(t)

    @staticmethod
    def _restore(kept):
        return kept.restore()
