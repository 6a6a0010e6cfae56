"""The policy operators from their definitions in 64 bits, on the CPU, and the error that a correct kernel can make.

Tolerances are worst-case sums of roundings.  Every function below is a sum of products, so the same function of the absolute
values is the magnitude M that each rounding scales with; u = finfo(type).eps / 2 is the largest relative error of a rounding.
"""
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def decay_reference(q, k, v, log_decay, state=None, start=None, scale=None, do=None, dfinal=None, magnitude=False):
    """(o, final) or, with do, (o, final, dq, dk, dv, dstate) as float64 CPU tensors; magnitude: of the absolute values"""
    def f(x):
        x = x.detach().double().cpu()
        return x.abs() if magnitude else x
    q, k, v = f(q), f(k), f(v)
    steps, envs, heads, dk = q.shape
    scale = dk ** -0.5 if scale is None else abs(scale) if magnitude else scale
    g = log_decay.detach().double().cpu().exp()[None, :, None, None]
    s = torch.zeros(envs, heads, dk, v.shape[3], dtype=torch.float64) if state is None else f(state).clone()
    cut = torch.zeros(steps + 1, envs, dtype=torch.bool)
    if start is not None:
        cut[:steps] = start.cpu() != 0
    cut = cut[:, :, None, None, None]
    o, dq = [], []
    do = None if do is None else f(do)
    for t in range(steps):
        s = torch.where(cut[t], torch.zeros_like(s), g * s) + k[t][..., :, None] * v[t][..., None, :]
        o.append(scale * (q[t][..., :, None] * s).sum(-2))
        if do is not None:
            dq.append(scale * (s * do[t][..., None, :]).sum(-1))
    o = torch.stack(o) if steps else q.new_zeros(0, envs, heads, v.shape[3])
    if do is None:
        return o, s
    d = torch.zeros_like(s) if dfinal is None else f(dfinal).clone()
    dks, dvs = [None] * steps, [None] * steps
    for t in reversed(range(steps)):
        d = d + scale * q[t][..., :, None] * do[t][..., None, :]
        dks[t] = (d * v[t][..., None, :]).sum(-1)
        dvs[t] = (d * k[t][..., :, None]).sum(-2)
        d = torch.where(cut[t], torch.zeros_like(d), g * d)
    return o, s, torch.stack(dq), torch.stack(dks), torch.stack(dvs), d


def decay_bounds(args, kw, dtype):
    """the largest error of each output: M times the roundings on the way to it.
    * In 32 bits: a sum of at most steps + 2 * 128 terms (u each, twice: products and sums), a power of the decay (an exponent
      of at most steps * |log_decay| rounded by u, the exponential by 2 u, once per step at the most: 4 u a step).
    * 16-bit inputs: the scores and the state inside a product are rounded to the type (u each, and one factor only in any
      product), tokens that enter the state are held in two parts of the type (u^2), three in bfloat16 (u^3).
    * The result is rounded to the type (states: float32)."""
    mags = decay_reference(*args, **kw, magnitude=True)
    refs = decay_reference(*args, **kw)
    steps, g = args[0].shape[0], float(args[3].detach().double().clamp(min=-80).abs().max())
    n32 = (2 * (steps + 256) + steps * (4 + g)) * U32
    u = half_step(dtype)
    out = []
    for i, (m, r) in enumerate(zip(mags, refs)):
        is_state = i in (1, 5)
        inner = 0.0 if dtype == torch.float32 else 2 * u if not is_state else 2 * u ** (2 if dtype == torch.float16 else 3)
        out.append((n32 + inner) * m + (U32 if is_state else u) * r.abs() + 1e-30)
    return refs, out


def norm_reference(x, weight, bias, eps, dy=None):
    x = x.detach().double().cpu()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if bias is None else bias.detach().double().cpu()
    mu = x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    h = (x - mu) * r
    y = h * w + b
    if dy is None:
        return (y,)
    dy = dy.detach().double().cpu()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    flat = x.shape[-1]
    return y, dx, (dy * h).reshape(-1, flat).sum(0), dy.reshape(-1, flat).sum(0)


def norm_bounds(x, weight, bias, eps, dy=None):
    """(references, largest errors).  All in units of the row's deviation: the row's sums take at most n = width / 32 + 32
    roundings in sequence, so a computed mean is off by n U mean|x| and a centred value by e = n U (|x| + mean|x|) rstd.  The
    centred second moment is then off by 2 mean(|h| e) + mean(e^2) <= 2 E + E^2 with E = rms(e) (rms(h) <= 1) and n U of its
    own, rstd by half of that, and h = c rstd by eh = e + |h| (E + E^2 / 2 + n U).  The rest follows term by term."""
    refs = norm_reference(x, weight, bias, eps, dy)
    dtype = x.dtype
    pdtype = weight.dtype if weight is not None else dtype
    xd = x.detach().double().cpu()
    width = xd.shape[-1]
    w = torch.ones(width, dtype=torch.float64) if weight is None else weight.detach().double().cpu().abs()
    b = torch.zeros(width, dtype=torch.float64) if bias is None else bias.detach().double().cpu().abs()
    mu = xd.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((xd - mu) ** 2).mean(-1, keepdim=True) + eps)
    h = ((xd - mu) * r).abs()
    nu = (width / 32 + 32) * U32
    e = nu * (xd.abs() + xd.abs().mean(-1, keepdim=True)) * r
    rms = (e * e).mean(-1, keepdim=True).sqrt()
    er = rms + rms * rms / 2 + nu  # rstd's relative error
    eh = 1.1 * (e + h * er)
    out = [w * eh + 4 * U32 * (h * w + b) + half_step(dtype) * refs[0].abs()]
    if dy is not None:
        d = dy.detach().double().cpu().abs()
        g = d * w
        mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
        mag = g + mean(g) + h * mean(g * h)
        out.append(r * (1.1 * (er + 2 * nu) * mag + 1.1 * (eh * mean(g * (h + eh)) + h * mean(g * eh)))
                   + half_step(dtype) * refs[1].abs())
        rows = xd.numel() // width
        cols = lambda t: t.reshape(-1, width).sum(0)  # noqa: E731
        out.append(cols(d * eh + (rows + 8) * U32 * d * h) + half_step(pdtype) * refs[2].abs())
        out.append((rows + 8) * U32 * cols(d) + half_step(pdtype) * refs[3].abs())
    return refs, [z + 1e-30 for z in out]


def assert_close(got, ref, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got - ref).abs()[bad].max()), float(bound[bad].min()))
