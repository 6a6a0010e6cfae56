"""A policy that remembers, for the device-resident rollouts of `urgym_amd.vec.URGymTorchVecEnv`.

No registered task observes a velocity (BallBalance: the paddle's angles and its offset to the ball), so one observation does
not say where the ball is going.  `MemoryPolicy` keeps, per env, what it has seen of the running episode in the state of
`urgym_amd.ops.decay_attention`:

* `step(obs, state, start)` -- one observation per env, inside a rollout, the state updated in place;
* `forward(obs, start, state)` -- a recorded rollout [steps, envs, ...] at once, differentiable, for training: the same
  answers as the steps gave, with the episodes that an autoreset packed into one time axis kept apart.

    env = URGymTorchVecEnv("URGym/BallBalance-v0", 4096); env.reset()
    policy = MemoryPolicy(6, 3).to(env.device)
    state = policy.initial_state(4096)
    rew, done, rec = env.rollout(policy, 64, state=state, record=True)
    actions, _ = policy(rec["obs"], rec["start"], rec["state"])        # with gradients
"""
import torch

from . import ops


class _Norm(torch.nn.Module):
    def __init__(self, width):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(width))
        self.bias = torch.nn.Parameter(torch.zeros(width))

    def forward(self, x):
        return ops.layer_norm(x, self.weight, self.bias)


class _Block(torch.nn.Module):
    def __init__(self, width, heads):
        super().__init__()
        self.heads = heads
        self.norm1, self.norm2 = _Norm(width), _Norm(width)
        self.qkv = torch.nn.Linear(width, 3 * width, bias=False)
        self.out = torch.nn.Linear(width, width, bias=False)
        self.up = torch.nn.Linear(width, 2 * width)
        self.down = torch.nn.Linear(2 * width, width)

    def forward(self, x, attend):
        qkv = self.qkv(self.norm1(x)).unflatten(-1, (3, self.heads, x.shape[-1] // self.heads))
        x = x + self.out(attend(*qkv.unbind(-3)).flatten(-2))
        return x + self.down(torch.nn.functional.silu(self.up(self.norm2(x))))


class MemoryPolicy(torch.nn.Module):
    """obs_dim -> act_dim with `layers` blocks of decay attention (`heads` heads) of the given width; the heads' horizons (steps
    until the decay has reached 1 / e) run from 2 to `horizon`."""

    has_memory = True  # URGymTorchVecEnv.rollout() steps it

    def __init__(self, obs_dim, act_dim, width=128, heads=4, layers=2, horizon=128.0):
        super().__init__()
        if heads < 1 or width % heads:
            raise ValueError(f"width {width} is not divisible into {heads} heads")
        if width // heads > ops.MAX_HEAD_DIM:
            raise ValueError(f"heads of {width // heads}: at most {ops.MAX_HEAD_DIM} (use more heads)")
        if not horizon >= 2:
            raise ValueError(f"horizon must be at least 2 steps, not {horizon}")
        self.heads, self.head_dim = heads, width // heads
        self.embed = torch.nn.Linear(obs_dim, width)
        self.blocks = torch.nn.ModuleList(_Block(width, heads) for _ in range(layers))
        self.norm = _Norm(width)
        self.head = torch.nn.Linear(width, act_dim)
        steps = 2.0 * (horizon / 2.0) ** (torch.arange(heads, dtype=torch.float32) / max(heads - 1, 1))
        self.register_buffer("log_decay", -1.0 / steps)

    def _apply(self, fn, *args, **kw):
        exact = self.log_decay
        super()._apply(fn, *args, **kw)
        if self.log_decay.dtype != exact.dtype:  # the weights' type is converted; decays of another type would be other horizons
            self.log_decay = exact.to(self.log_decay.device)
        return self

    def initial_state(self, envs):
        """one state per block: nothing remembered"""
        return [torch.zeros(envs, self.heads, self.head_dim, self.head_dim, dtype=torch.float32, device=self.log_decay.device) for _ in self.blocks]

    def _run(self, obs, attend):
        x = self.embed(obs.to(self.embed.weight.dtype))
        for i, block in enumerate(self.blocks):
            x = block(x, lambda q, k, v: attend(i, q, k, v))
        return self.head(self.norm(x))

    @torch.no_grad()
    def step(self, obs, state, start=None):
        """obs [envs, obs_dim], state of `initial_state` (updated in place), start [envs] (set where an episode begins):
        actions [envs, act_dim]"""
        return self._run(obs, lambda i, q, k, v: ops.decay_attention_step(q, k, v, self.log_decay, state[i], start=start,
                                                                          state_out=state[i])[0])

    def forward(self, obs, start=None, state=None):
        """obs [steps, envs, obs_dim], start [steps, envs], state before the first step (None: nothing remembered):
        (actions [steps, envs, act_dim], the state after the last step)"""
        final = []

        def attend(i, q, k, v):
            o, s = ops.decay_attention(q, k, v, self.log_decay, None if state is None else state[i], start)
            final.append(s)
            return o

        return self._run(obs, attend), final


__all__ = ["MemoryPolicy"]
