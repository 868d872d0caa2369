"""The gated recurrence of the recurrent agent over a rollout [steps, environments, features], with its gradient: `acx_scan_forward` /
`acx_scan_backward` (csrc/acx_scan.hip); a block of the agent made of it and its end (block_norm), over a rollout and, in one launch,
for a single step (`acx_block_step`, csrc/acx_block.hip).  The reference's agent has no memory (ac_solver/agents/ppo_agent.py:11-109)."""
import torch

from ac_solver import _acx
from ac_solver.agents import _tensors as T
from ac_solver.agents import activation8
from ac_solver.agents.block_norm import MAX_WIDTH, block_output_backward, block_output_forward


def _operands(candidate, gate, reset, state):
    candidate = T.activation(candidate, "candidate")
    if candidate.dim() != 3:
        raise ValueError(f"candidate has to be [steps, rows, features], not {tuple(candidate.shape)}")
    gate = T.activation(gate, "gate", like=candidate, shape=candidate.shape)
    steps, rows, width = candidate.shape
    if steps < 1:
        raise ValueError("a scan needs at least one step")
    if reset is not None:
        reset = T.flags(reset, "reset", (steps, rows), candidate.device)
    if state is not None:
        state = T.plain(state, "state", (rows, width), candidate.device)
    T.require_gpu(candidate)
    return candidate, gate, reset, state


def gated_scan_forward(candidate, gate, reset=None, state=None, save=True):
    """The forward pass alone -> (hidden, last_state, bounds); `bounds` is what `gated_scan_backward` needs besides the operands, None
    without `save`."""
    candidate, gate, reset, state = _operands(candidate, gate, reset, state)
    steps, rows, width = candidate.shape
    dev = candidate.device
    hidden = torch.empty((steps, rows, width), dtype=candidate.dtype, device=dev)
    last = torch.empty((rows, width), dtype=torch.float32, device=dev)
    bounds = torch.empty(_acx.lib.acx_scan_bounds_bytes(steps, rows, width) // 4, dtype=torch.float32, device=dev) if save else None
    code = T.DTYPES[candidate.dtype]
    work = T.scratch(_acx.lib.acx_scan_workspace_bytes(steps, rows, width, code), dev)
    with T.on_device_of(candidate):
        _acx.check(_acx.lib.acx_scan_forward(candidate.data_ptr(), candidate.stride(0), candidate.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1), code,
                                             T.ptr(reset), T.ptr(state), steps, rows, width, hidden.data_ptr(), last.data_ptr(), T.ptr(bounds), T.ptr(work),
                                             0 if work is None else work.numel(), T.stream_of(candidate)), "acx_scan_forward")
    return hidden, last, bounds


def gated_scan_backward(d_hidden, d_last, candidate, gate, reset, bounds, want_state=True, out=None):
    """Gradients of candidate, gate and initial state from those of hidden and last state (`d_last` may be None).  `out`: two tensors
    [steps, rows, features] to write the first two into (slices of a projection's gradient, say).  -> (d_candidate, d_gate, d_state or None)"""
    candidate, gate, reset, _ = _operands(candidate, gate, reset, None)
    steps, rows, width = candidate.shape
    dev = candidate.device
    d_hidden = T.activation(d_hidden, "d_hidden", like=candidate, shape=candidate.shape)
    d_last = None if d_last is None else T.plain(d_last, "d_last", (rows, width), dev)
    bounds = T.plain(bounds, "bounds", (_acx.lib.acx_scan_bounds_bytes(steps, rows, width) // 4,), dev)
    if out is None:
        dc, dz = (torch.empty((steps, rows, width), dtype=candidate.dtype, device=dev) for _ in range(2))
    else:
        dc, dz = out
        for t, name in ((dc, "out[0]"), (dz, "out[1]")):
            if T.activation(t, name, like=candidate, shape=candidate.shape) is not t:
                raise ValueError(f"{name} has to have a contiguous last axis")
    d_state = torch.empty((rows, width), dtype=torch.float32, device=dev) if want_state else None
    code = T.DTYPES[candidate.dtype]
    work = T.scratch(_acx.lib.acx_scan_workspace_bytes(steps, rows, width, code), dev)
    with T.on_device_of(candidate):
        _acx.check(_acx.lib.acx_scan_backward(candidate.data_ptr(), candidate.stride(0), candidate.stride(1), gate.data_ptr(), gate.stride(0), gate.stride(1),
                                              d_hidden.data_ptr(), d_hidden.stride(0), d_hidden.stride(1), code, T.ptr(reset), bounds.data_ptr(), T.ptr(d_last), steps, rows,
                                              width, dc.data_ptr(), dc.stride(0), dc.stride(1), dz.data_ptr(), dz.stride(0), dz.stride(1), T.ptr(d_state), T.ptr(work),
                                              0 if work is None else work.numel(), T.stream_of(candidate)), "acx_scan_backward")
    return dc, dz, d_state


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, candidate, gate, reset, state):
        hidden, last, bounds = gated_scan_forward(candidate, gate, reset, state, save=any(ctx.needs_input_grad))
        ctx.save_for_backward(candidate, gate, reset, bounds)
        ctx.set_materialize_grads(False)
        return hidden, last

    @staticmethod
    @T.once
    def backward(ctx, d_hidden, d_last):
        candidate, gate, reset, bounds = ctx.saved_tensors
        if d_hidden is None:
            if d_last is None:
                return None, None, None, None
            d_hidden = torch.zeros((), dtype=candidate.dtype, device=candidate.device).expand(candidate.shape)
        dc, dz, d_state = gated_scan_backward(d_hidden, d_last, candidate, gate, reset, bounds, ctx.needs_input_grad[3])
        return dc if ctx.needs_input_grad[0] else None, dz if ctx.needs_input_grad[1] else None, None, d_state


def gated_scan(candidate, gate, reset=None, state=None):
    """Along the steps t of candidate, gate [steps, rows, features] (float32, bfloat16 or float16; slices of a projection as they are):

        f = sigmoid(gate[t]);  h[t] = f * h[t - 1] + (1 - f) * candidate[t]

    with h[t - 1] replaced by zero where `reset` [steps, rows] (bool) says that an episode starts at step t, and h[-1] = `state`
    [rows, features] float32, or zero.  The recurrence runs in float32 whatever the type of the activations.
    -> (hidden [steps, rows, features] of the activations' type, last state [rows, features] float32); both differentiable (once) with
    respect to candidate, gate and state."""
    return _GatedScan.apply(candidate, gate, reset, state)


class _RecurrentBlock(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, projected, reset, state, weight, scale, next_weight, eps):
        width = x.shape[-1]
        candidate, gate, out_gate = (projected[..., k * width:(k + 1) * width] for k in range(3))
        save = any(ctx.needs_input_grad)
        hidden, last, bounds = gated_scan_forward(candidate, gate, reset, state, save=save)
        new, u, stats = block_output_forward(x, hidden, out_gate, weight, scale, next_weight, eps, save=save)
        if save:
            # (autograd packs x and projected itself inside checkpoint8; hidden is nobody's input)
            ctx.packed = activation8.packing() and hidden.numel() >= activation8.MIN_VALUES
            kept = activation8.pack8(hidden) if ctx.packed else (hidden,)
            ctx.save_for_backward(x, projected, reset, weight, scale, next_weight, bounds, stats, *kept)
        ctx.set_materialize_grads(False)
        return new, u, last

    @staticmethod
    @T.once
    def backward(ctx, d_new, d_u, d_last):
        if d_new is None and d_u is None and d_last is None:
            return (None,) * 8
        x, projected, reset, weight, scale, next_weight, bounds, stats, *kept = ctx.saved_tensors
        hidden = activation8.unpack8(*kept, x.dtype) if ctx.packed else kept[0]
        width = x.shape[-1]
        thirds = lambda t: [t[..., k * width:(k + 1) * width] for k in range(3)]  # noqa: E731
        candidate, gate, out_gate = thirds(projected)
        d_projected = torch.empty(projected.shape, dtype=projected.dtype, device=projected.device)
        d_candidate, d_gate, d_out_gate = thirds(d_projected)
        dx, d_hidden, _, dw, ds, dn = block_output_backward(d_new, d_u, x, hidden, out_gate, weight, scale, next_weight, stats, d_gate_out=d_out_gate)
        _, _, d_state = gated_scan_backward(d_hidden, d_last, candidate, gate, reset, bounds, want_state=ctx.needs_input_grad[3], out=(d_candidate, d_gate))
        grads = (dx, d_projected, None, d_state, dw, ds, dn)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,)


def recurrent_block(x, projected, state, weight, scale=None, next_weight=None, reset=None, eps=1e-6):
    """A block of the recurrent agent over a rollout, differentiable (once): with candidate, gate, output gate = the three thirds of projected
    [steps, rows, 3 width] (a projection of the block's normalised input),

        hidden, last = gated_scan(candidate, gate, reset, state);  new, u = block_output(x, hidden, output gate, weight, scale, next_weight, eps)

    -> (new, u, last): the residual stream behind the block, its norm for the next one (None without `next_weight`), the last state.  The
    gradient of `projected` is written in place by the two operators, without a copy of its thirds."""
    if not isinstance(x, torch.Tensor) or x.dim() != 3:
        raise ValueError("x has to be [steps, rows, features]")
    T.activation(projected, "projected", like=T.activation(x, "x"), shape=x.shape[:-1] + (3 * x.shape[-1],))
    return _RecurrentBlock.apply(x, projected, reset, state, weight, scale, next_weight, eps)


def recurrent_step(x, projected, state, weight, scale=None, next_weight=None, reset=None, next_state=None, eps=1e-6):
    """A whole block for ONE step of the environments in one launch (rollouts; no gradient): with candidate, gate, output gate = the
    three thirds of projected [rows, 3 width],

        h = gated_scan of one step from `state` [rows, width] float32 (zero where `reset` [rows] (bool) says that an episode starts)
        new, u = block_output(x, h, output gate, weight, scale, next_weight, eps)

    x and projected of one type (float32, bfloat16 or float16); h stays float32.  `next_state`: where the new state goes, `state` itself for
    in place; None: a new tensor.  -> (new, u, next_state); u is None without `next_weight`."""
    x = T.activation(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x has to be [rows, features], not {tuple(x.shape)}")
    rows, width = x.shape
    if width > MAX_WIDTH:
        raise ValueError(f"rows of up to {MAX_WIDTH} features are handled, not {width}")
    if not eps >= 0.0:
        raise ValueError(f"eps has to be a number of at least 0, not {eps}")
    dev = x.device
    projected = T.activation(projected, "projected", like=x, shape=(rows, 3 * width))
    state = T.plain(state, "state", (rows, width), dev)
    weight = T.plain(weight, "weight", (width,), dev)
    scale = None if scale is None else T.plain(scale, "scale", (width,), dev)
    next_weight = None if next_weight is None else T.plain(next_weight, "next_weight", (width,), dev)
    if reset is not None:
        reset = T.flags(reset, "reset", (rows,), dev)
    if next_state is not None and T.plain(next_state, "next_state", (rows, width), dev) is not next_state:
        raise ValueError("next_state has to be contiguous")
    T.require_gpu(x)
    if next_state is None:
        next_state = torch.empty_like(state)
    new = torch.empty((rows, width), dtype=x.dtype, device=dev)
    u = None if next_weight is None else torch.empty((rows, width), dtype=x.dtype, device=dev)
    if rows and width:
        with T.on_device_of(x):
            _acx.check(_acx.lib.acx_block_step(x.data_ptr(), x.stride(0), projected.data_ptr(), projected.stride(0), T.DTYPES[x.dtype], T.ptr(reset), state.data_ptr(),
                                               weight.data_ptr(), T.ptr(scale), T.ptr(next_weight), eps, rows, width, next_state.data_ptr(), new.data_ptr(), T.ptr(u),
                                               T.stream_of(x)), "acx_block_step")
    return new, u, next_state
