"""The norms in front of and behind a block of the recurrent agent, with the block's gate and residual scale: `acx_block_forward` /
`acx_block_backward` (csrc/acx_block.hip).  The reference's agent has no such layers (ac_solver/agents/ppo_agent.py:11-109)."""
import torch

from ac_solver import _acx
from ac_solver.agents import _tensors as T

MAX_WIDTH = 4096


def _rows(t):
    """[..., width] -> [rows, width] with one stride between rows (a copy only where the leading axes have none in common)"""
    return t.reshape(-1, t.shape[-1])


def _operands(x, y, gate, weight, scale, next_weight, eps):
    x = T.activation(x, "x")
    if x.dim() < 1:
        raise ValueError("x has to have a feature axis")
    width = x.shape[-1]
    if width > MAX_WIDTH:
        raise ValueError(f"rows of up to {MAX_WIDTH} features are handled, not {width}")
    if not eps >= 0.0:
        raise ValueError(f"eps has to be a number of at least 0, not {eps}")
    if y is not None:
        y = T.activation(y, "y", like=x, shape=x.shape)
        weight = T.plain(weight, "weight", (width,), x.device)
    if gate is not None:
        gate = T.activation(gate, "gate", like=x, shape=x.shape)
    if scale is not None:
        scale = T.plain(scale, "scale", (width,), x.device)
    if next_weight is not None:
        next_weight = T.plain(next_weight, "next_weight", (width,), x.device)
    T.require_gpu(x)
    return x, y, gate, weight, scale, next_weight


def block_output_forward(x, y, gate, weight, scale=None, next_weight=None, eps=1e-6, save=True):
    """The forward pass alone -> (new, u, stats); `stats` [rows, 2] is what `block_output_backward` needs besides the operands, None without
    `save`; u is None without `next_weight`, new is None without `y`."""
    x, y, gate, weight, scale, next_weight = _operands(x, y, gate, weight, scale, next_weight, eps)
    width, dev = x.shape[-1], x.device
    x2, y2, g2 = _rows(x) if x.numel() else x, None if y is None or not x.numel() else _rows(y), None if gate is None or not x.numel() else _rows(gate)
    new = None if y is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
    u = None if next_weight is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
    rows = x.numel() // width if width else 0
    stats = torch.empty((rows, 2), dtype=torch.float32, device=dev) if save else None
    if rows:
        with T.on_device_of(x):
            _acx.check(_acx.lib.acx_block_forward(x2.data_ptr(), x2.stride(0), T.ptr(y2), 0 if y2 is None else y2.stride(0), T.ptr(g2), 0 if g2 is None else g2.stride(0),
                                                  T.DTYPES[x.dtype], T.ptr(weight), T.ptr(scale), T.ptr(next_weight), eps, rows, width, T.ptr(new), T.ptr(u), T.ptr(stats),
                                                  T.stream_of(x)), "acx_block_forward")
    return new, u, stats


def block_output_backward(d_new, d_u, x, y, gate, weight, scale, next_weight, stats, d_gate_out=None):
    """Gradients from those of new and u (each may be None) -> (d_x, d_y, d_gate, d_weight, d_scale, d_next_weight), None for an operand that
    is None.  `d_gate_out`: a tensor of the gate's shape to write its gradient into (a slice of a projection's gradient, say)."""
    x, y, gate, weight, scale, next_weight = _operands(x, y, gate, weight, scale, next_weight, 0.0)
    width, dev = x.shape[-1], x.device
    if d_u is not None and next_weight is None:
        raise ValueError("a gradient of u without next_weight")
    grads = [None if t is None else T.activation(t, name, like=x, shape=x.shape) for t, name in ((d_new, "d_new"), (d_u, "d_u"))]
    rows = x.numel() // width if width else 0
    stats = T.plain(stats, "stats", (rows, 2), dev)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dy = None if y is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
    dg = None if gate is None else (torch.empty(x.shape, dtype=x.dtype, device=dev) if d_gate_out is None else d_gate_out)
    weights = torch.empty((3, width), dtype=torch.float32, device=dev)
    if rows:
        x2, y2, g2, n2, u2 = (None if t is None else _rows(t) for t in (x, y, gate, *grads))
        dg2 = None
        if dg is not None:
            T.activation(dg, "d_gate_out", like=x, shape=x.shape)
            dg2 = dg.view(-1, width)  # (raises where the rows have no common stride: the result has to land in the caller's tensor)
            if width > 1 and dg2.stride(1) != 1:
                raise ValueError("d_gate_out has to have a contiguous last axis")
        code = T.DTYPES[x.dtype]
        work = T.scratch(_acx.lib.acx_block_workspace_bytes(rows, width, code), dev)
        st = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
        with T.on_device_of(x):
            _acx.check(_acx.lib.acx_block_backward(x2.data_ptr(), st(x2), T.ptr(y2), st(y2), T.ptr(g2), st(g2), T.ptr(n2), st(n2), T.ptr(u2), st(u2), code, T.ptr(weight),
                                                   T.ptr(scale), T.ptr(next_weight), stats.data_ptr(), rows, width, dx.data_ptr(), T.ptr(dy), T.ptr(dg2), st(dg2),
                                                   weights.data_ptr(), work.data_ptr(), work.numel(), T.stream_of(x)), "acx_block_backward")
    else:
        weights.zero_()
    return (dx, dy, dg, weights[0] if y is not None else None, weights[1] if scale is not None and y is not None else None,
            weights[2] if next_weight is not None else None)


class _BlockOutput(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, weight, scale, next_weight, eps):
        new, u, stats = block_output_forward(x, y, gate, weight, scale, next_weight, eps, save=any(ctx.needs_input_grad))
        ctx.save_for_backward(x, y, gate, weight, scale, next_weight, stats)
        ctx.set_materialize_grads(False)
        return new, u

    @staticmethod
    @T.once
    def backward(ctx, d_new, d_u):
        if d_new is None and d_u is None:
            return (None,) * 7
        grads = block_output_backward(d_new, d_u, *ctx.saved_tensors)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,)


def block_output(x, y, gate, weight, scale=None, next_weight=None, eps=1e-6):
    """The end of a block in one pass over the rows (last axis of x, y, gate: float32, bfloat16 or float16, up to 4096 features; weights
    float32 [width]):

        new = x + scale * silu(gate) * rms(y) * weight;  u = rms(new) * next_weight;  rms(v) = v / sqrt(mean(v^2) + eps)

    `gate` None: no gate; `scale` None: 1; `next_weight` None: no norm in front of a next block (u is None).  Computed in float32 and rounded
    once: u comes from the unrounded new.  -> (new, u), differentiable (once) with respect to all tensors; the gradients of the weights are
    summed over the rows in a fixed order."""
    return _BlockOutput.apply(x, y, gate, weight, scale, next_weight, eps)


def block_input(x, weight, eps=1e-6):
    """u = rms(x) * weight: the norm in front of the first block (see block_output for types and sizes)"""
    return _BlockOutput.apply(x, None, None, None, None, weight, eps)[1]
