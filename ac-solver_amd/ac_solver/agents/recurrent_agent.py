"""An agent with a memory (`--recurrent` of ac_solver.agents.ppo): a shared trunk of gated recurrent blocks over the steps of an episode, with
the actor and the critic as linear heads.  The reference's agent (ac_solver/agents/ppo_agent.py:11-109: two tanh MLPs over the current
observation) stays the default; it chooses a move from the presentation alone, this one also from the way that led to it.

    x = encoder(obs);  u = rms(x) norm
    for each block:  candidate, gate, output gate = projection(u)
                     h[t] = f h[t - 1] + (1 - f) candidate[t],  f = sigmoid(gate[t]),  h = 0 where an episode starts
                     x += scale * silu(output gate) * rms(h) weight;  u = rms(x) (the next block's norm, the last one's for the heads)

Over a rollout the recurrence is one scan (recurrence.recurrent_block), a step of the environments costs one launch per block beside the
projections (recurrence.recurrent_step)."""
import numpy as np
import torch
from torch import nn
from torch.distributions import Categorical
from torch.nn import functional as F

from ac_solver.agents import activation8
from ac_solver.agents.block_norm import block_input
from ac_solver.agents.ppo_agent import Linear, initialize_layer
from ac_solver.agents.recurrence import recurrent_block, recurrent_step

MAX_WIDTH = 4096  # of block_norm
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


class Block(nn.Module):
    def __init__(self, width, forget_bias=2.0):
        super().__init__()
        self.norm = nn.Parameter(torch.ones(width))  # in front of the projection
        self.projection = initialize_layer(Linear(width, 3 * width), 1.0)
        self.weight = nn.Parameter(torch.ones(width))  # of the norm behind the recurrence
        self.scale = nn.Parameter(torch.full((width,), 0.5))
        with torch.no_grad():  # sigmoid(2): a memory of about eight steps to begin with
            self.projection.bias[width:2 * width] = forget_bias


class RecurrentAgent(nn.Module):
    """`dtype`: of the activations in the trunk ("float32" or "bfloat16"; parameters, states and heads are float32).  `checkpoint_8bit`: a
    training pass keeps its activations in 8 bits for the backward pass (activation8)."""

    is_recurrent = True

    def __init__(self, envs, width=256, blocks=2, dtype="float32", checkpoint_8bit=False):
        super().__init__()
        if width < 1 or blocks < 1:
            raise ValueError("a recurrent agent has at least one block of at least one feature")
        if width > MAX_WIDTH:
            raise ValueError(f"blocks of up to {MAX_WIDTH} features are handled, not {width}")
        self.width, self.dtype, self.checkpoint_8bit = int(width), DTYPES[dtype], bool(checkpoint_8bit)
        input_dim = int(np.prod(envs.single_observation_space.shape))
        self.encoder = initialize_layer(Linear(input_dim, self.width))
        self.blocks = nn.ModuleList(Block(self.width) for _ in range(blocks))
        self.norm = nn.Parameter(torch.ones(self.width))
        self.actor = initialize_layer(Linear(self.width, int(envs.single_action_space.n)), 0.01)
        self.critic = initialize_layer(Linear(self.width, 1), 1.0)

    def initial_state(self, rows, device=None):
        """[blocks, rows, width] float32 zeros"""
        return torch.zeros((len(self.blocks), rows, self.width), device=device or self.norm.device)

    def _linear(self, layer, x):
        if self.checkpoint_8bit and torch.is_grad_enabled():
            return activation8.linear8(x, layer.weight, layer.bias)
        if x.dtype == torch.float32:
            return layer(x.reshape(-1, x.shape[-1])).view(*x.shape[:-1], -1)
        return F.linear(x, layer.weight.to(x.dtype), layer.bias.to(x.dtype))

    def _norm_behind(self, k):
        return self.blocks[k + 1].norm if k + 1 < len(self.blocks) else self.norm

    def features(self, obs, reset, state):
        """obs [steps, rows, ...], reset [steps, rows] bool, state [blocks, rows, width] -> (features [steps, rows, width], last states)"""
        steps, rows = obs.shape[:2]
        x = self._linear(self.encoder, obs.reshape(steps, rows, -1).to(self.dtype))
        u = block_input(x, self.blocks[0].norm)
        last = []
        for k, b in enumerate(self.blocks):
            x, u, h = recurrent_block(x, self._linear(b.projection, u), state[k], b.weight, b.scale, self._norm_behind(k), reset=reset)
            last.append(h)
        return u, torch.stack(last)

    @torch.no_grad()
    def step_features(self, obs, reset, state, next_state):
        """one step: obs [rows, ...], reset [rows] bool; the states go from `state` to `next_state` (the same tensor: in place)"""
        x = self._linear(self.encoder, obs.reshape(obs.shape[0], -1).to(self.dtype))
        u = block_input(x, self.blocks[0].norm)
        for k, b in enumerate(self.blocks):
            x, u, _ = recurrent_step(x, self._linear(b.projection, u), state[k], b.weight, b.scale, self._norm_behind(k), reset=reset, next_state=next_state[k])
        return u

    @torch.no_grad()
    def act(self, obs, reset, state):
        """a rollout step -> (action, its log-probability, value); `state` moves on in place"""
        u = self.step_features(obs, reset, state, state).float()
        dist = Categorical(logits=self.actor(u), validate_args=False)
        action = dist.sample()
        return action, dist.log_prob(action), self.critic(u).flatten()

    @torch.no_grad()
    def get_value(self, obs, reset, state):
        """the value of observations that are not acted on yet: the states stay where they are"""
        return self.critic(self.step_features(obs, reset, state, torch.empty_like(state)).float()).flatten()

    def evaluate(self, obs, actions, reset, state):
        """a rollout again, from the states in front of its first step -> (log-probability, entropy, value) of all steps [steps * rows]"""
        if self.checkpoint_8bit and torch.is_grad_enabled():
            with activation8.checkpoint8():
                u, _ = self.features(obs, reset, state)
        else:
            u, _ = self.features(obs, reset, state)
        u = u.reshape(-1, self.width).float()
        dist = Categorical(logits=self.actor(u), validate_args=False)
        return dist.log_prob(actions.reshape(-1)), dist.entropy(), self.critic(u).flatten()
