"""The policy operators of urgym_amd.ops as a user's program calls them: layer norm, attention with a per-head decay over recorded
rollouts, and its one-token form inside a rollout.  Each case runs in plain torch operations, or, with `own`, through the package.
"""
import math

import torch

own = False
DEVICE = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


def _norm(rows, width, dtype, param, train):
    return {"op": "layer_norm", "rows": rows, "width": width, "dtype": dtype, "param": param, "train": train}


def _step(envs, heads, dk, dv, dtype):
    return {"op": "decay_step", "envs": envs, "heads": heads, "dk": dk, "dv": dv, "dtype": dtype}


def _seq(steps, envs, heads, dk, dv, dtype, train, episode, carry, fused):
    """episode: the mean episode length, 0 for no episode starts inside; carry: a state from before is continued;
    fused: q, k and v are slices of one projection's output"""
    return {"op": "decay_seq", "steps": steps, "envs": envs, "heads": heads, "dk": dk, "dv": dv, "dtype": dtype,
            "train": train, "episode": episode, "carry": carry, "fused": fused}


def listed():
    return [
        # one rollout step of a 256-wide policy over BallBalance's 4096 envs: latency counts
        {"name": "norm_rollout_4096x256_bf16", **_norm(4096, 256, "bfloat16", "float32", False)},
        # CubesGrasp's 17 observations (an odd width) over a recorded rollout of 25 steps x 8192 envs
        {"name": "norm_obs_204800x17_f32", **_norm(204800, 17, "float32", "float32", True)},
        # the policy's width over 500 steps (BallBalance's time limit) x 1024 envs, with its gradients
        {"name": "norm_train_512000x256_bf16", **_norm(512000, 256, "bfloat16", "float32", True)},
        # few wide rows: the norm before a wide policy's last layer, odd sizes
        {"name": "norm_wide_4097x5000_f16", **_norm(4097, 5000, "float16", "float16", True)},
        # a single env (make() without num_envs): latency only
        {"name": "step_1x4x32_f32", **_step(1, 4, 32, 32, "float32")},
        # BallBalance's 4096 envs: the state's bytes count
        {"name": "step_4096x4x64_bf16", **_step(4096, 4, 64, 64, "bfloat16")},
        # an odd number of envs, heads whose key and value widths differ
        {"name": "step_1000x3x48x80_f16", **_step(1000, 3, 48, 80, "float16")},
        # one long recorded trajectory read back into the memory: few heads, a long axis
        {"name": "seq_8192x1x8x64_bf16", **_seq(8192, 1, 8, 64, 64, "bfloat16", False, 0, False, False)},
        # CubesPush: 50-step episodes of 4096 envs in full precision, the state carried from the rollout before
        {"name": "seq_train_50x4096x4x32_f32", **_seq(50, 4096, 4, 32, 32, "float32", True, 30, True, False)},
        # BallBalance's 500 steps of 1024 envs, many episodes packed in the time axis: the large training pass
        {"name": "seq_train_500x1024x4x64_bf16", **_seq(500, 1024, 4, 64, 64, "bfloat16", True, 100, False, False)},
        # a small ragged batch: nothing is a multiple of anything
        {"name": "seq_train_333x37x5x24x40_f16", **_seq(333, 37, 5, 24, 40, "float16", True, 15, True, False)},
        # Box-v0's 200 steps, wide heads, q | k | v from one projection: values of a recorded rollout
        {"name": "seq_200x256x2x128_bf16", **_seq(200, 256, 2, 128, 128, "bfloat16", False, 100, True, True)},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "decay_step", "decay_seq", "decay_seq"])
    dtype = rng.choice(sorted(TYPES))
    if op == "layer_norm":
        width = _log_int(rng, 4, 8192)
        rows = _log_int(rng, 1, min(400000, 60000000 // width))
        return _norm(rows, width, dtype, rng.choice([dtype, "float32"]), rng.random() < 0.6)
    heads = rng.choice([1, 2, 3, 4, 5, 8])
    dk = rng.choice([8, 16, 24, 32, 48, 64, 65, 80, 96, 128, rng.randint(4, 128)])
    dv = dk if rng.random() < 0.6 else rng.choice([8, 20, 32, 33, 64, 72, 128, rng.randint(4, 128)])
    if op == "decay_step":
        return _step(_log_int(rng, 1, min(8192, 60000000 // (heads * dk * dv))), heads, dk, dv, dtype)
    steps = _log_int(rng, 1, 4096)
    most = min(4096, 400000000 // (steps * steps * heads), 64000000 // (steps * heads * max(dk, dv)),
               100000000 // (heads * dk * dv))
    envs = _log_int(rng, 1, max(1, most))
    episode = rng.choice([0, 0, 3, 15, 50, 200])
    return _seq(steps, envs, heads, dk, dv, dtype, rng.random() < 0.6, episode, rng.random() < 0.5, rng.random() < 0.3)


def _starts(steps, envs, episode, gen):
    """episode starts [steps, envs]: episode lengths uniform in 1 .. 2 episode - 1, the first one cut anywhere"""
    lengths = torch.randint(1, 2 * episode, (steps + 1, envs), generator=gen, device=DEVICE)
    at = torch.cumsum(lengths, 0) - torch.randint(0, episode + 1, (1, envs), generator=gen, device=DEVICE)
    start = torch.zeros(steps, envs, dtype=torch.bool, device=DEVICE)
    inside = (at >= 0) & (at < steps)
    env = torch.arange(envs, device=DEVICE).expand_as(at)
    start[at[inside], env[inside]] = True
    return start


def _decays(heads):
    """horizons from 2 steps to 128, spread over the heads"""
    horizon = torch.logspace(1, 7, heads, base=2.0, dtype=torch.float64) if heads > 1 else torch.tensor([32.0], dtype=torch.float64)
    return torch.log1p(-1.0 / horizon).to(torch.float32).to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32)

    dtype = TYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "layer_norm":
        rows, width, param = case["rows"], case["width"], TYPES[case["param"]]
        st["x"] = (normal(rows, width) * 1.5 + 0.5 * normal(rows, 1) + 0.3).to(dtype)
        st["weight"] = (1.0 + 0.1 * normal(width)).to(param)
        st["bias"] = (0.1 * normal(width)).to(param)
        if case["train"]:
            st["dy"] = normal(rows, width).to(dtype)
            for name in ("x", "weight", "bias"):
                st[name].requires_grad_()
        return st
    heads, dk, dv, envs = case["heads"], case["dk"], case["dv"], case["envs"]
    st["log_decay"] = _decays(heads)
    if case["op"] == "decay_step":
        st["q"], st["k"] = normal(envs, heads, dk).to(dtype), normal(envs, heads, dk).to(dtype)
        st["v"] = normal(envs, heads, dv).to(dtype)
        st["state"] = 3.0 * normal(envs, heads, dk, dv)
        st["start"] = torch.rand(envs, generator=gen, device=DEVICE) < 0.05
        st["state_out"] = torch.empty_like(st["state"])
        return st
    steps = case["steps"]
    if case["fused"]:
        qkv = normal(steps, envs, heads * (2 * dk + dv)).to(dtype)
        q, k, v = qkv.split([heads * dk, heads * dk, heads * dv], -1)
        st["q"], st["k"], st["v"] = q.unflatten(-1, (heads, dk)), k.unflatten(-1, (heads, dk)), v.unflatten(-1, (heads, dv))
    else:
        st["q"], st["k"] = normal(steps, envs, heads, dk).to(dtype), normal(steps, envs, heads, dk).to(dtype)
        st["v"] = normal(steps, envs, heads, dv).to(dtype)
    st["start"] = _starts(steps, envs, case["episode"], gen) if case["episode"] else None
    st["state"] = 3.0 * normal(envs, heads, dk, dv) if case["carry"] else None
    if case["train"]:
        st["do"] = normal(steps, envs, heads, dv).to(dtype)
        st["dstate"] = normal(envs, heads, dk, dv)
        for name in ("q", "k", "v", "state"):
            if st[name] is not None:
                st[name] = st[name].detach().requires_grad_()
    return st


# ---- the plain forms ----

def _plain_norm(st):
    x = st["x"].float()
    w, b = st["weight"].float(), st["bias"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    hat = centred * rstd
    y = (hat * w + b).to(st["x"].dtype)
    if not st["case"]["train"]:
        return y
    dy = st["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    return y, dx.to(st["x"].dtype), (dy * hat).sum(0).to(st["weight"].dtype), dy.sum(0).to(st["bias"].dtype)


def _plain_step(st):
    scale = st["case"]["dk"] ** -0.5
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    old = torch.where(st["start"][:, None, None, None], torch.zeros_like(st["state"]), st["state"])
    new = old * torch.exp(st["log_decay"])[:, None, None] + k[..., :, None] * v[..., None, :]
    o = scale * (q[..., :, None] * new).sum(-2)
    return o.to(st["q"].dtype), new


def _batched(x):
    """[steps, envs, heads, d] in 32 bits as [envs, heads, steps, d]"""
    return x.float().permute(1, 2, 0, 3).contiguous()


def _timed(x, dtype):
    return x.permute(2, 0, 1, 3).contiguous().to(dtype)


def _plain_seq(st):
    case = st["case"]
    steps, envs, heads = case["steps"], case["envs"], case["heads"]
    dtype, scale = st["q"].dtype, case["dk"] ** -0.5
    q, k, v = _batched(st["q"]), _batched(st["k"]), _batched(st["v"])
    at = torch.arange(steps, device=q.device)
    start = torch.zeros(steps, envs, dtype=torch.bool, device=q.device) if st["start"] is None else st["start"]
    episode = torch.cumsum(start.int(), 0).t().contiguous()  # [envs, steps]
    apart = (at[:, None] - at[None, :]).float()
    power = torch.exp(st["log_decay"][:, None, None] * apart.clamp(min=0))  # [heads, steps, steps]
    seen = (apart >= 0) & (episode[:, :, None] == episode[:, None, :])
    weight = torch.where(seen[:, None], scale * power, torch.zeros((), device=q.device))  # [envs, heads, steps, steps]
    reach = torch.where((episode == 0)[:, None], torch.exp(st["log_decay"][:, None] * (at + 1).float()),
                        torch.zeros((), device=q.device))[..., None]  # of the carried state, [envs, heads, steps, 1]
    last = torch.where((episode == episode[:, -1:])[:, None], torch.exp(st["log_decay"][:, None] * (steps - 1 - at).float()),
                       torch.zeros((), device=q.device))[..., None]  # of each step on the final state
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * weight
    o = torch.matmul(scores, v)
    final = torch.matmul((last * k).transpose(-1, -2).contiguous(), v)
    if case["carry"]:
        s0 = st["state"].float()
        o = o + scale * reach * torch.matmul(q, s0)
        final = final + reach[:, :, -1:] * s0
    o = _timed(o, dtype)
    if not case["train"]:
        return o, final
    do, dfinal = _batched(st["do"]), st["dstate"]
    dv = torch.matmul(scores.transpose(-1, -2).contiguous(), do) + last * torch.matmul(k, dfinal)
    dscores = torch.matmul(do, v.transpose(-1, -2).contiguous()) * weight
    dq = torch.matmul(dscores, k)
    dk = torch.matmul(dscores.transpose(-1, -2).contiguous(), q) + last * torch.matmul(v, dfinal.transpose(-1, -2).contiguous())
    out = [o, final, _timed(dq, dtype), _timed(dk, dtype), _timed(dv, dtype)]
    if case["carry"]:
        dq = dq + scale * reach * torch.matmul(do, s0.transpose(-1, -2).contiguous())
        out[2] = _timed(dq, dtype)
        out.append(scale * torch.matmul((reach * q).transpose(-1, -2).contiguous(), do) + reach[:, :, -1:] * dfinal)
    return out


# ---- the package's calls ----

def _own(st):
    from urgym_amd import ops
    case = st["case"]
    if case["op"] == "layer_norm":
        y = ops.layer_norm(st["x"], st["weight"], st["bias"], eps=EPS)
        if not case["train"]:
            return y
        return (y, *torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"]))
    if case["op"] == "decay_step":
        return ops.decay_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"], start=st["start"],
                                        state_out=st["state_out"])
    o, final = ops.decay_attention(st["q"], st["k"], st["v"], st["log_decay"], state=st["state"], start=st["start"])
    if not case["train"]:
        return o, final
    leaves = [st["q"], st["k"], st["v"]] + ([st["state"]] if case["carry"] else [])
    return [o, final, *torch.autograd.grad((o, final), leaves, (st["do"], st["dstate"]))]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        op = state["case"]["op"]
        return _plain_norm(state) if op == "layer_norm" else _plain_step(state) if op == "decay_step" else _plain_seq(state)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "layer_norm":
        n, param = case["rows"] * case["width"], 4 if case["param"] == "float32" else 2
        if case["train"]:  # x and dy in, y and dx out, weight and bias in, their gradients out
            return {"bytes": 4 * n * size + 4 * case["width"] * param, "flops": 22 * n}
        return {"bytes": 2 * n * size + 2 * case["width"] * param, "flops": 8 * n}
    heads, dk, dv, envs = case["heads"], case["dk"], case["dv"], case["envs"]
    states = envs * heads * dk * dv
    if case["op"] == "decay_step":
        return {"bytes": 8 * states + envs * heads * 2 * (dk + dv) * size + envs, "flops": 5 * states}
    tokens = case["steps"] * envs * heads
    flags = case["steps"] * envs if case["episode"] else 0
    moved = tokens * 2 * (dk + dv) * size + flags + 4 * states * (2 if case["carry"] else 1)
    flops = 4 * tokens * dk * dv
    if case["train"]:  # do and the final state's gradient in; dq, dk, dv and the first state's gradient out
        moved += tokens * (2 * dk + 2 * dv) * size + 4 * states * (2 if case["carry"] else 1)
        flops += 10 * tokens * dk * dv
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits ----

def _exact_norm(st):
    x, w, b = (st[n].detach().double() for n in ("x", "weight", "bias"))
    width = x.shape[-1]
    mu = x.sum(-1, keepdim=True) / width
    var = ((x - mu) ** 2).sum(-1, keepdim=True) / width
    sigma = torch.sqrt(var + EPS)
    y = (x - mu) / sigma * w + b
    if not st["case"]["train"]:
        return y
    dy = st["dy"].double()
    # y_i = w_i c_i / sigma + b_i with c = x - mu: through c and through sigma, then through mu
    dc = dy * w / sigma - (x - mu) * ((dy * w * (x - mu)).sum(-1, keepdim=True) / (width * sigma ** 3))
    dx = dc - dc.sum(-1, keepdim=True) / width
    return y, dx, (dy * (x - mu) / sigma).sum(0), dy.sum(0)


def _exact_step(st):
    gamma = st["log_decay"].double().exp()[None, :, None, None]
    s = st["state"].double().clone()
    s[st["start"]] = 0
    s = gamma * s + torch.einsum("nhk,nhv->nhkv", st["k"].double(), st["v"].double())
    return torch.einsum("nhk,nhkv->nhv", st["q"].double(), s) / math.sqrt(st["case"]["dk"]), s


def _exact_seq(st):
    case = st["case"]
    steps, envs, heads, dk, dv = (case[n] for n in ("steps", "envs", "heads", "dk", "dv"))
    f64 = torch.float64
    gamma = st["log_decay"].double().exp()[None, :, None, None]
    scale = 1.0 / math.sqrt(dk)
    device = st["q"].device
    keep = None if st["start"] is None else (~st["start"]).double()[:, :, None, None, None]
    s = torch.zeros(envs, heads, dk, dv, dtype=f64, device=device) if st["state"] is None else st["state"].detach().double().clone()
    o = torch.empty(steps, envs, heads, dv, dtype=f64, device=device)
    dq = torch.empty(steps, envs, heads, dk, dtype=f64, device=device) if case["train"] else None
    for t in range(steps):
        q, k, v = (st[n][t].detach().double() for n in "qkv")
        s = s * gamma if keep is None else s * (gamma * keep[t])
        s.addcmul_(k[..., :, None], v[..., None, :])
        o[t] = scale * torch.matmul(q[..., None, :], s)[..., 0, :]
        if case["train"]:
            dq[t] = scale * torch.matmul(s, st["do"][t].double()[..., :, None])[..., 0]
    if not case["train"]:
        return o, s
    d = st["dstate"].double().clone()
    dks, dvs = torch.empty_like(dq), torch.empty_like(o)
    for t in reversed(range(steps)):
        q, k, v = (st[n][t].detach().double() for n in "qkv")
        d.addcmul_(scale * q[..., :, None], st["do"][t].double()[..., None, :])
        dks[t] = torch.matmul(d, v[..., :, None])[..., 0]
        dvs[t] = torch.matmul(k[..., None, :], d)[..., 0, :]
        d = d * gamma if keep is None else d * (gamma * keep[t])
    return [o, s, dq, dks, dvs] + ([d] if case["carry"] else [])


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(st) if case["op"] == "layer_norm" else _exact_step(st) if case["op"] == "decay_step" else _exact_seq(st)
