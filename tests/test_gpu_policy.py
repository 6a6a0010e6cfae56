"""A policy with memory on the env's stream: stepped through a rollout, then trained on the recorded rollout, whose episodes
the autoreset packed into one time axis -- the operators of urgym_amd.ops as they are used together."""
import numpy as np
import pytest
import torch



def test_policy_refusals():
    from urgym_amd.policy import MemoryPolicy
    for kw in (dict(width=30, heads=4), dict(width=260, heads=2), dict(heads=0), dict(horizon=1.0)):
        with pytest.raises(ValueError):
            MemoryPolicy(6, 3, **kw)
    p = MemoryPolicy(6, 3, width=32, heads=4, layers=3)
    assert [tuple(s.shape) for s in p.initial_state(5)] == [(5, 4, 8, 8)] * 3
    assert torch.allclose(p.log_decay, -1.0 / torch.tensor([2.0, 8.0, 32.0, 128.0]))
    with pytest.raises(ValueError, match="no CPU fallback"):
        p(torch.zeros(4, 5, 6))


def test_rollout_steps_a_policy_with_memory_cpu(monkeypatch):
    """rollout()'s bookkeeping with a scripted simulator: starts after reset and after each done, the state handed through,
    what is recorded, and a policy without memory served as before"""
    from contextlib import nullcontext
    from urgym_amd.vec import URGymTorchVecEnv
    env = object.__new__(URGymTorchVecEnv)
    n = 3
    env.torch, env.num_envs, env.device, env._fresh = torch, n, torch.device("cpu"), True
    env.obs = torch.zeros(n, 2, dtype=torch.float64)
    env.terminated, env.truncated = torch.zeros(n, dtype=torch.uint8), torch.zeros(n, dtype=torch.uint8)
    env.low, env.high = torch.full((1,), -0.1), torch.full((1,), 0.1)
    env.stream_context, env._enter, env._leave = nullcontext, lambda: None, lambda cur: None
    dones = torch.tensor([[0, 1, 0], [0, 0, 1], [1, 0, 0], [0, 0, 0]], dtype=torch.uint8)
    t = [0]

    def step(act):
        env.obs += 1.0
        env.terminated.copy_(dones[t[0] % 4])
        t[0] += 1
        env._fresh = False
        return env.obs, act[:, 0].double(), env.terminated, env.truncated, None
    env.step = step

    class Memory:
        seen = []

        def initial_state(self, envs):
            return [torch.zeros(envs)]

        def step(self, obs, state, start):
            self.seen.append(start.tolist())
            state[0].copy_(torch.where(start != 0, torch.zeros_like(state[0]), state[0]) + 1)
            return state[0][:, None].clone()
    p = Memory()
    rew, done, rec = env.rollout(p, 4, record=True)
    assert p.seen == [[1, 1, 1], [0, 1, 0], [0, 0, 1], [1, 0, 0]] and rec["start"].tolist() == p.seen
    assert done.tolist() == [1, 1, 1, 0] and rec["terminated"].tolist() == dones.tolist()
    assert rec["obs"][:, 0, 0].tolist() == [0.0, 1.0, 2.0, 3.0] and rec["action"].shape == (4, 3, 1)
    assert rec["action"].max() <= 0.1 + 1e-6 and not rec["state"][0].any()
    state = [torch.tensor([5.0, 6.0, 7.0])]
    assert len(env.rollout(p, 1, state=state)) == 2 and state[0].tolist() == [6.0, 7.0, 8.0] and p.seen[-1] == [0, 0, 0]
    rew, done, rec = env.rollout(lambda obs: obs[:, :1], 2, record=True)
    assert rec["state"] is None and rew.shape == (2,)
    with pytest.raises(TypeError):
        env.rollout(lambda obs: obs[:, :1], 2, state=state)


@pytest.mark.gpu
@pytest.mark.parametrize("env_id,obs_dim,act_dim", [("URGym/BallBalance-v0", 6, 3), ("URGym/CubesGrasp-v0", 17, 9)])
def test_rollout_then_training_on_it(built, env_id, obs_dim, act_dim):
    from urgym_amd.policy import MemoryPolicy
    from urgym_amd.vec import URGymTorchVecEnv
    torch.manual_seed(0)
    n, T = 16, 30  # longer than CubesGrasp's 20-step limit: every env autoresets inside
    env = URGymTorchVecEnv(env_id, n, seed=3)
    env.reset()
    policy = MemoryPolicy(obs_dim, act_dim, width=64, heads=2, layers=2).to(env.device)
    state = policy.initial_state(n)
    rew, done, rec = env.rollout(policy, T, state=state, record=True)
    torch.cuda.current_stream().wait_stream(env.stream)
    assert int(done.sum()) > 0 and bool(rec["start"][0].all())
    assert torch.equal(rec["start"][1:], rec["terminated"][:-1] | rec["truncated"][:-1])
    assert torch.allclose(rec["reward"].sum(1), rew)
    actions, final = policy(rec["obs"], rec["start"], rec["state"])
    # the steps and the sequence are the same function; two layers of 64-term products in float32, inputs of size 1
    inside = torch.maximum(torch.minimum(actions.detach(), env.high), env.low)
    assert float((inside - rec["action"]).abs().max()) < 1e-4
    for a, b in zip(final, state):
        assert float((a.detach() - b).abs().max()) < 1e-3 * float(b.abs().max())
    # the next rollout goes on from there
    _, _, rec2 = env.rollout(policy, 3, state=state, record=True)
    assert torch.equal(rec2["start"][0], rec["terminated"][-1] | rec["truncated"][-1])
    assert all(not torch.equal(a, b) for a, b in zip(rec2["state"], state))
    # gradients: every parameter has one, and along a direction it is the difference of the loss
    weight = torch.randn_like(actions)
    params = [p for p in policy.parameters()]
    grads = torch.autograd.grad((actions * weight).sum(), params)
    assert all(torch.isfinite(g).all() and g.abs().sum() > 0 for g in grads)
    gen = torch.Generator(device=env.device).manual_seed(1)
    step = 1e-2
    direction = [torch.randn(p.shape, generator=gen, device=p.device) * p.detach().std().clamp(min=0.05) for p in params]
    ends = []
    with torch.no_grad():
        for sign in (1, -2, 1):
            for p, d in zip(params, direction):
                p.add_(sign * step * d)
            if sign != 1 or not ends:
                ends.append(float((policy(rec["obs"], rec["start"], rec["state"])[0].double() * weight).sum()))
    slope = (ends[0] - ends[1]) / (2 * step)
    want = float(sum((g.double() * d).sum() for g, d in zip(grads, direction)))
    scale = float(sum((g.double() * d).pow(2).sum() for g, d in zip(grads, direction)) ** 0.5)
    assert abs(slope - want) < 0.05 * max(abs(want), scale), (slope, want, scale)
    env.close()
    assert np.isfinite(ends).all()
