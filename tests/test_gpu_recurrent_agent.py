"""The recurrent agent (ac_solver/agents/recurrent_agent.py): its operators together, as the trainer uses them -- a rollout step by step, the
same rollout as one pass, its gradients against a float64 autograd of the formulas, 8-bit checkpoints, and the training loop itself."""
from types import SimpleNamespace

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def spaces(in_dim, n_act):
    return SimpleNamespace(single_observation_space=SimpleNamespace(shape=(in_dim,)), single_action_space=SimpleNamespace(n=n_act))


def make_agent(in_dim=50, n_act=12, width=48, blocks=2, seed=0, **kw):
    import torch

    from ac_solver.agents.recurrent_agent import RecurrentAgent

    torch.manual_seed(seed)
    agent = RecurrentAgent(spaces(in_dim, n_act), width, blocks, **kw).cuda()
    with torch.no_grad():
        for p in agent.parameters():  # nothing at its special initial value
            p.add_(torch.randn_like(p) * 0.1)
    return agent


def rollout(T, N, in_dim, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    obs = torch.randint(-2, 3, (T, N, in_dim), device="cuda", generator=g).float()
    start = torch.rand((T, N), device="cuda", generator=g) < 0.15
    return obs, start, torch.randint(0, 12, (T, N), device="cuda", generator=g)


def plain_features(agent, obs, start, state):
    """the agent's formulas in float64, step by step; -> (features [T, N, width], last states), differentiable in the float64 copies `p` of the
    parameters"""
    import torch

    p = {k: v.detach().double().requires_grad_() for k, v in agent.named_parameters()}
    rms = lambda v: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    x = obs.double() @ p["encoder.weight"].T + p["encoder.bias"]
    D, K = agent.width, len(agent.blocks)
    last = []
    for k in range(K):
        q = f"blocks.{k}."
        proj = (rms(x) * p[q + "norm"]) @ p[q + "projection.weight"].T + p[q + "projection.bias"]
        c, z, g = proj[..., :D], proj[..., D:2 * D], proj[..., 2 * D:]
        f, h, hs = torch.sigmoid(z), state[k].double(), []
        for t in range(obs.shape[0]):
            h = f[t] * h.masked_fill(start[t, :, None], 0.0) + (1 - f[t]) * c[t]
            hs.append(h)
        last.append(h)
        x = x + p[q + "scale"] * g * torch.sigmoid(g) * rms(torch.stack(hs)) * p[q + "weight"]
    return rms(x) * p["norm"], torch.stack(last), p


@pytest.mark.parametrize("width,blocks", [(48, 2), (33, 1), (256, 3)])
def test_a_pass_and_its_steps_and_the_formulas_agree(width, blocks):
    """float32: some 30 T relative roundings of 2^-24 pass through a block and the norms keep values of order one: 1e-4 leaves a factor of ten"""
    import torch

    T, N = 40, 7
    agent = make_agent(width=width, blocks=blocks)
    obs, start, actions = rollout(T, N, 50, 1)
    state0 = torch.randn_like(agent.initial_state(N))
    with torch.no_grad():
        u, last = agent.features(obs, start, state0)
        want, want_last, _ = plain_features(agent, obs, start, state0)
        state = state0.clone()
        steps = torch.stack([agent.step_features(obs[t], start[t], state, state) for t in range(T)])
    top = float(want.abs().max())
    assert float((u - want).abs().max()) < 1e-4 * top and float((steps - want).abs().max()) < 1e-4 * top
    assert float((last - want_last).abs().max()) < 1e-4 * float(want_last.abs().max()) and float((state - last).abs().max()) < 1e-4 * top
    # acting gives what evaluating the actions gives, and a value that is looked at does not move the memory
    memory, kept = state0.clone(), []
    for t in range(T):
        before = memory.clone()
        v = agent.get_value(obs[t], start[t], memory)
        assert torch.equal(memory, before)
        a, lp, val = agent.act(obs[t], start[t], memory)
        assert torch.equal(v, val)
        kept.append((a, lp, val))
    a, lp, val = (torch.stack([k[i] for k in kept]) for i in range(3))
    with torch.no_grad():
        lp2, ent, val2 = agent.evaluate(obs, a, start, state0)
    assert float((lp2.view(T, N) - lp).abs().max()) < 1e-3 and float((val2.view(T, N) - val).abs().max()) < 1e-3 and ent.shape == (T * N,)


def loss_of(lp, ent, val):
    return (lp * 0.7 - 0.01 * ent + (val - 0.3) ** 2).mean()


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_gradients_against_the_formulas(dtype, checkpoint):
    """relative to each parameter's largest gradient: float32 a few hundred roundings; bfloat16 2^-9 for each of the ~10 tensors a value passes through;
    8-bit checkpoints 2^-8 of a block's largest value for each kept tensor, which enters a gradient as noise of random sign"""
    import torch

    from ac_solver.agents.recurrent_agent import RecurrentAgent  # noqa: F401

    T, N = 40, 24
    agent = make_agent(width=64, dtype=dtype, checkpoint_8bit=checkpoint)
    obs, start, actions = rollout(T, N, 50, 2)
    state0 = torch.randn_like(agent.initial_state(N))
    loss = loss_of(*agent.evaluate(obs, actions, start, state0))
    grads = torch.autograd.grad(loss, list(agent.parameters()))
    u, _, p = plain_features(agent, obs, start, state0)
    u = u.reshape(-1, agent.width)
    logp = torch.log_softmax(u @ p["actor.weight"].T + p["actor.bias"], -1)
    val = (u @ p["critic.weight"].T + p["critic.bias"]).flatten()
    want = torch.autograd.grad(loss_of(logp.gather(1, actions.reshape(-1, 1)).flatten(), -(logp.exp() * logp).sum(-1), val), list(p.values()))
    tol = {("float32", False): 2e-3, ("float32", True): 0.1, ("bfloat16", False): 0.1, ("bfloat16", True): 0.15}[dtype, checkpoint]
    for (name, _), g, w in zip(p.items(), grads, want):
        assert g.dtype == torch.float32 and g.shape == w.shape
        assert float((g - w).abs().max()) <= tol * float(w.abs().max()), (name, float((g - w).abs().max()), float(w.abs().max()))


def test_checkpoints_take_less_memory():
    import torch

    used = {}
    for checkpoint in (False, True):
        agent = make_agent(width=256, checkpoint_8bit=checkpoint)
        obs, start, actions = rollout(64, 256, 50, 3)
        state0 = agent.initial_state(256)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = agent.evaluate(obs, actions, start, state0)
        used[checkpoint] = torch.cuda.memory_allocated() - before
        torch.autograd.grad(loss_of(*out), list(agent.parameters()))
        del out
    # per block and value in float32: x, the normed input, three thirds of the projection and the hidden value, 24 bytes; 6.2 with 8 bits; the
    # states between segments and the heads' float32 features stay
    assert used[True] < 0.45 * used[False], used


@pytest.mark.parametrize("kw", [{}, {"recurrent_dtype": "bfloat16"}, {"checkpoint_8bit": "true"}])
def test_the_training_loop_trains_it(golden_json, kw):
    import torch
    from torch.optim import Adam

    from ac_solver.agents.recurrent_agent import RecurrentAgent
    from ac_solver.agents.training import ppo_training_loop
    from ac_solver.envs.vec_env import ACVecEnv
    from tests.conftest import ms_pool_generator_order
    from tests.test_gpu_ppo import _args

    L, N, T, H = 18, 8, 24, 10
    easy = np.zeros(2 * L, np.int8)
    easy[:2], easy[L] = [1, 2], 2
    initial_states = [easy.tolist()] + [list(p) for p in ms_pool_generator_order(golden_json("ms_pool.json"))[:7]]
    args = _args(num_envs=N, num_steps=T, total_timesteps=N * T * 3, horizon_length=H, update_epochs=2, num_minibatches=4, seed=5, recurrent="true",
                 recurrent_width=32, target_kl=10.0, **kw)
    device = torch.device("cuda", 0)
    torch.manual_seed(args.seed)
    envs = ACVecEnv(np.asarray(initial_states, np.int8), horizon_length=H, obs_dtype="float32", clip_rewards=(args.min_rew, args.max_rew), record_actions=True,
                    final_info=False, device=device)
    agent = RecurrentAgent(envs, args.recurrent_width, args.recurrent_blocks, args.recurrent_dtype, args.checkpoint_8bit).to(device)
    before = [p.detach().clone() for p in agent.parameters()]
    seen = []
    inner = agent.evaluate

    def evaluate(obs, actions, reset, state):
        seen.append((reset.clone(), state.clone()))
        return inner(obs, actions, reset, state)

    agent.evaluate = evaluate
    rec = {"solved": set(), "unsolved": set(range(N))}
    log = []
    stats = ppo_training_loop(envs, args, device, Adam(agent.parameters(), lr=args.learning_rate, eps=args.epsilon), agent, list(range(N)), rec, {}, set(range(N)),
                              initial_states, progress=False, rollout_log=log)
    assert len(log) == 3 and all(np.isfinite(stats[k]) for k in ("losses/value_loss", "losses/policy_loss", "losses/entropy_loss", "losses/approx_kl"))
    # every parameter moved; the unchanged weights give the rollout's own probabilities (a pass and its steps differ by roundings)
    assert all(not torch.equal(a, b.detach()) for a, b in zip(before, agent.parameters()))
    assert stats["debug/ratio0_maxdev"] < (1e-3 if args.recurrent_dtype == "float32" else 1e-2)
    # the first update starts from empty memories at the start of episodes, a later one from what the rollout before it left
    first = [s for s in seen[:len(seen) // 3]]
    assert all(bool(r[0].all()) and not bool(m.any()) for r, m in first)
    assert any(bool(m.any()) for _, m in seen[len(seen) // 3:])
    # an episode's start is marked where one ended the step before, by reaching the goal or at the horizon (every H steps at the latest)
    starts = torch.cat([r for r, _ in seen[-4:]], dim=1)
    assert all(bool(starts[t:t + H].any(0).all()) for t in range(T - H + 1))


def test_the_command_trains_it(tmp_path, monkeypatch):
    from ac_solver.agents.ppo import train_ppo

    monkeypatch.chdir(tmp_path)
    stats = train_ppo(["--recurrent", "--recurrent-width", "64", "--fixed-init-state", "--num-envs", "8", "--num-steps", "20", "--total-timesteps", "480",
                       "--horizon-length", "15", "--checkpoint-8bit"])
    assert stats["charts/global_step"] == 480 and np.isfinite(stats["losses/value_loss"])
