"""Which policies URGymTorchVecEnv.rollout() steps as policies with memory, with a scripted simulator."""
from contextlib import nullcontext

import pytest
import torch

from urgym_amd.policy import MemoryPolicy
from urgym_amd.vec import URGymTorchVecEnv


def _env(n=3):
    env = object.__new__(URGymTorchVecEnv)
    env.torch, env.num_envs, env.device, env._fresh = torch, n, torch.device("cpu"), True
    env.obs = torch.zeros(n, 2, dtype=torch.float64)
    env.terminated, env.truncated = torch.zeros(n, dtype=torch.uint8), torch.zeros(n, dtype=torch.uint8)
    env.low, env.high = torch.full((1,), -1.0), torch.full((1,), 1.0)
    env.stream_context, env._enter, env._leave = nullcontext, lambda: None, lambda cur: None

    def step(act):
        env.obs += 1.0
        env._fresh = False
        return env.obs, act[:, 0].double(), env.terminated, env.truncated, None
    env.step = step
    return env


class Recurrent(torch.nn.Module):
    """a module of someone else's, called as policy(obs), with methods of the same names"""
    has_memory = False

    def __init__(self):
        super().__init__()
        self.calls = []

    def initial_state(self, batch):
        return [torch.zeros(batch)]

    def step(self, obs, state, start):
        self.calls.append("step")
        state[0] += 1
        return obs[:, :1] * 0

    def forward(self, obs):
        self.calls.append("call")
        return obs[:, :1] * 0


def test_a_module_with_methods_of_these_names_is_called_as_before():
    plain = Recurrent()
    del Recurrent.has_memory
    try:
        assert len(_env().rollout(plain, 2)) == 2 and plain.calls == ["call"] * 2
        _, _, rec = _env().rollout(plain, 1, record=True)
        assert plain.calls == ["call"] * 3 and rec["state"] is None
    finally:
        Recurrent.has_memory = False
    _env().rollout(plain, 1)
    assert plain.calls == ["call"] * 4


def test_a_module_that_says_so_or_is_given_a_state_is_stepped():
    p = Recurrent()
    p.has_memory = True
    _, _, rec = _env().rollout(p, 2, record=True)
    assert p.calls == ["step"] * 2 and len(rec["state"]) == 1
    p, state = Recurrent(), [torch.zeros(3)]
    _env().rollout(p, 2, state=state)
    assert p.calls == ["step"] * 2 and state[0].tolist() == [2.0] * 3
    assert MemoryPolicy.has_memory
    with pytest.raises(TypeError):
        _env().rollout(lambda obs: obs[:, :1], 1, state=state)
