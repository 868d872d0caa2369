"""The gated recurrence of the recurrent agent over a rollout [steps, environments, features], with its gradient: `acx_scan_forward` /
`acx_scan_backward` (csrc/acx_scan.hip); a block of the agent made of it and its end (block_norm), over a rollout and, in one launch,
for a single step (`acx_block_step`, csrc/acx_block.hip).  The reference's agent has no memory (ac_solver/agents/ppo_agent.py:11-109).

Arguments that do not fit raise TypeError (types) or ValueError (shapes, places, values) before anything is launched.
Kernels go to the current stream of the tensors' device."""
from ac_solver.agents import activation8
from ac_solver.agents._ops import ops


def gated_scan(candidate, gate, reset=None, state=None):
    """Along the steps t of candidate, gate [steps, rows, features] (float32, bfloat16 or float16; slices of a projection as they are):

        f = sigmoid(gate[t]);  h[t] = f * h[t - 1] + (1 - f) * candidate[t]

    with h[t - 1] replaced by zero where `reset` [steps, rows] (bool) says that an episode starts at step t, and h[-1] = `state`
    [rows, features] float32, or zero.  The recurrence runs in float32 whatever the type of the activations.
    -> (hidden [steps, rows, features] of the activations' type, last state [rows, features] float32); both differentiable (once) with
    respect to candidate, gate and state."""
    return ops.gated_scan(candidate, gate, reset, state)


def gated_scan_forward(candidate, gate, reset=None, state=None, save=True):
    """The forward pass alone, outside autograd -> (hidden, last_state, bounds); `bounds` is what `gated_scan_backward` needs besides the
    operands, None without `save`."""
    return ops.gated_scan_forward(candidate, gate, reset, state, save)


def gated_scan_backward(d_hidden, d_last, candidate, gate, reset, bounds, want_state=True, out=None):
    """Gradients of candidate, gate and initial state from those of hidden and last state (`d_last` may be None).  `out`: two tensors
    [steps, rows, features] to write the first two into (slices of a projection's gradient, say; not over an operand).
    -> (d_candidate, d_gate, d_state or None)"""
    return ops.gated_scan_backward(d_hidden, d_last, candidate, gate, reset, bounds, want_state, *((None, None) if out is None else out))


def recurrent_block(x, projected, state, weight, scale=None, next_weight=None, reset=None, eps=1e-6):
    """A block of the recurrent agent over a rollout, differentiable (once): with candidate, gate, output gate = the three thirds of projected
    [steps, rows, 3 width] (a projection of the block's normalised input),

        hidden, last = gated_scan(candidate, gate, reset, state);  new, u = block_output(x, hidden, output gate, weight, scale, next_weight, eps)

    -> (new, u, last): the residual stream behind the block, its norm for the next one (None without `next_weight`), the last state.  The
    gradient of `projected` is written in place by the two operators, without a copy of its thirds; inside activation8.checkpoint8 the hidden
    values are kept in 8 bits."""
    return ops.recurrent_block(x, projected, reset, state, weight, scale, next_weight, eps, activation8.packing() and x.numel() >= activation8.MIN_VALUES)


def recurrent_step(x, projected, state, weight, scale=None, next_weight=None, reset=None, next_state=None, eps=1e-6):
    """A whole block for ONE step of the environments in one launch (rollouts; no gradient): with candidate, gate, output gate = the
    three thirds of projected [rows, 3 width],

        h = gated_scan of one step from `state` [rows, width] float32 (zero where `reset` [rows] (bool) says that an episode starts)
        new, u = block_output(x, h, output gate, weight, scale, next_weight, eps)

    x and projected of one type (float32, bfloat16 or float16); h stays float32.  `next_state`: where the new state goes, `state` itself for
    in place; None: a new tensor.  -> (new, u, next_state); u is None without `next_weight`."""
    return ops.recurrent_step(x, projected, state, weight, scale, next_weight, reset, next_state, eps)
