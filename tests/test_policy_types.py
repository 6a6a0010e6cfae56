"""MemoryPolicy in types other than float32."""
import copy

import pytest
import torch

from urgym_amd.policy import MemoryPolicy


def test_decays_stay_float32():
    """the horizons that were asked for, whatever type the weights are converted to: 1 / 5.04 rounded to bfloat16 is another horizon"""
    p = MemoryPolicy(6, 3, width=32, heads=4, horizon=100.0)
    want = p.log_decay.clone()
    for convert in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.bfloat16().float(), lambda m: m.to("cpu", torch.float16),
                    lambda m: copy.deepcopy(m).double(), lambda m: torch.nn.Sequential(m).half()[0]):
        c = convert(copy.deepcopy(p))
        assert c.log_decay.dtype == torch.float32 and torch.equal(c.log_decay, want)
        assert torch.equal(c.state_dict()["log_decay"], want)
    other = MemoryPolicy(6, 3, width=32, heads=4, horizon=7.0).half()
    other.load_state_dict(p.half().state_dict())
    assert torch.equal(other.log_decay, want)
    for default in (torch.float64, torch.bfloat16):
        torch.set_default_dtype(default)
        try:
            assert torch.equal(MemoryPolicy(6, 3, width=32, heads=4, horizon=100.0).log_decay, want)
        finally:
            torch.set_default_dtype(torch.float32)
    empty = p.to("meta")
    assert empty.log_decay.is_meta and empty.to_empty(device="cpu").log_decay.dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("width,heads,envs", [(64, 2, 5), (256, 4, 300)])
def test_steps_and_sequence_agree_in_16_bits(built, dtype, width, heads, envs):
    """the token steps, the recorded rollout at once, and the same network in float32: in each layer's some 12 roundings to the type, each
    of half a step of its vector's norm, and none amplified more than 4 times (norms before every block): 2 layers of 12, 4 u each"""
    torch.manual_seed(1)
    exact = MemoryPolicy(6, 3, width=width, heads=heads, layers=2, horizon=50.0)
    policy = copy.deepcopy(exact).to("cuda", dtype)
    exact.load_state_dict({n: t.float() for n, t in policy.cpu().state_dict().items()})
    policy, exact = policy.cuda(), exact.cuda()
    obs = torch.randn(70, envs, 6).cuda().to(dtype)
    start = (torch.rand(70, envs) < 0.03).cuda()
    state, steps = policy.initial_state(envs), []
    for t in range(70):
        steps.append(policy.step(obs[t], state, start[t]))
    actions, final = policy(obs, start)
    wanted, states = exact(obs.float(), start)
    assert actions.dtype == dtype and all(s.dtype == torch.float32 for s in final)
    tol = 2 * 12 * 4 * torch.finfo(dtype).eps / 2

    def apart(a, b):
        return float((a.double() - b.double()).norm() / b.double().norm())
    assert apart(actions, wanted) < tol and apart(torch.stack(steps), wanted) < tol
    for a, b, c in zip(final, state, states):
        assert apart(a, c) < tol and apart(b, c) < tol
    grads = torch.autograd.grad((actions.float() * torch.randn_like(wanted)).sum(), list(policy.parameters()))
    assert all(g.dtype == dtype and torch.isfinite(g).all() and g.abs().sum() > 0 for g in grads)
