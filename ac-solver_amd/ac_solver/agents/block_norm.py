"""The norms in front of and behind a block of the recurrent agent, with the block's gate and residual scale: `acx_block_forward` /
`acx_block_backward` (csrc/acx_block.hip).  The reference's agent has no such layers (ac_solver/agents/ppo_agent.py:11-109)."""
from ac_solver.agents._ops import ops


def block_output(x, y, gate, weight, scale=None, next_weight=None, eps=1e-6):
    """The end of a block in one pass over the rows (last axis of x, y, gate: float32, bfloat16 or float16, up to 4096 features; weights
    float32 [width]):

        new = x + scale * silu(gate) * rms(y) * weight;  u = rms(new) * next_weight;  rms(v) = v / sqrt(mean(v^2) + eps)

    `gate` None: no gate; `scale` None: 1; `next_weight` None: no norm in front of a next block (u is None).  Computed in float32 and rounded
    once: u comes from the unrounded new.  -> (new, u), differentiable (once) with respect to all tensors; the gradients of the weights are
    summed over the rows in a fixed order."""
    return ops.block_output(x, y, gate, weight, scale, next_weight, eps)


def block_input(x, weight, eps=1e-6):
    """u = rms(x) * weight: the norm in front of the first block (see block_output for types and sizes)"""
    return ops.block_output(x, None, None, None, None, weight, eps)[1]


def block_output_forward(x, y, gate, weight, scale=None, next_weight=None, eps=1e-6, save=True):
    """The forward pass alone, outside autograd -> (new, u, stats); `stats` [rows, 2] is what `block_output_backward` needs besides the operands,
    None without `save`; u is None without `next_weight`, new is None without `y`."""
    return ops.block_output_forward(x, y, gate, weight, scale, next_weight, eps, save)


def block_output_backward(d_new, d_u, x, y, gate, weight, scale, next_weight, stats, d_gate_out=None):
    """Gradients from those of new and u (each may be None) -> (d_x, d_y, d_gate, d_weight, d_scale, d_next_weight), None for an operand that
    is None.  `d_gate_out`: a tensor of the gate's shape to write its gradient into (a slice of a projection's gradient, say; not
    over an operand)."""
    return ops.block_output_backward(d_new, d_u, x, y, gate, weight, scale, next_weight, stats, d_gate_out)
