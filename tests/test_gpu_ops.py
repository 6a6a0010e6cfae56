"""The policy operators on the GPU against their definitions in 64 bits (tests/ops_reference.py, which also derives the
tolerances): sizes from one token to several hundred, odd widths, strides, episode starts anywhere, infinities and NaN in
episodes that a token must not see, zero lengths, streams, graphs, and repeated calls."""
import ctypes

import pytest
import torch

from ops_reference import assert_close, decay_bounds, decay_reference, norm_bounds

pytestmark = pytest.mark.gpu
DEV = "cuda"
ALL = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops(built):
    from urgym_amd import ops
    return ops


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _decays(heads):
    return torch.log1p(-1.0 / torch.logspace(0.5, 6, heads, base=2.0)) if heads > 1 else torch.tensor([-0.1])


def _case(steps, envs, heads, dk, dv, dtype, starts=0.0, carry=False, seed=0):
    gen = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    q, k, v = (r(steps, envs, heads, d).to(dtype).to(DEV) for d in (dk, dk, dv))
    state = (3 * r(envs, heads, dk, dv)).to(DEV) if carry else None
    start = (torch.rand(steps, envs, generator=gen) < starts).to(DEV) if starts else None
    do, dfinal = r(steps, envs, heads, dv).to(dtype).to(DEV), r(envs, heads, dk, dv).to(DEV)
    return q, k, v, _decays(heads).to(DEV), state, start, do, dfinal


def _grads(ops, q, k, v, g, state, start, do, dfinal, **kw):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([state.detach().requires_grad_()] if state is not None else [])
    o, final = ops.decay_attention(*leaves[:3], g, leaves[3] if state is not None else None, start, **kw)
    return [o, final, *torch.autograd.grad((o, final), leaves, (do, dfinal))]


SIZES = [  # steps, envs, heads, dk, dv, starts, carry
    (1, 1, 1, 1, 1, 0.0, False), (1, 3, 2, 32, 32, 0.5, True), (2, 2, 1, 17, 33, 0.0, True), (15, 5, 3, 24, 40, 0.2, True),
    (16, 2, 2, 64, 64, 0.0, False), (17, 4, 1, 65, 31, 0.1, True), (31, 3, 2, 128, 128, 0.05, True), (32, 2, 4, 32, 16, 0.0, True),
    (33, 7, 2, 8, 128, 0.3, False), (64, 2, 2, 128, 40, 0.02, True), (95, 1, 5, 48, 80, 1.0, True), (127, 6, 1, 64, 96, 0.01, True),
    (300, 1, 2, 96, 32, 0.0, True), (777, 2, 1, 32, 64, 0.004, True),
]


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s[:5])))
def test_decay_attention(ops, size, dtype):
    q, k, v, g, state, start, do, dfinal = _case(*size[:5], dtype, *size[5:], seed=size[0])
    got = _grads(ops, q, k, v, g, state, start, do, dfinal)
    refs, bounds = decay_bounds((q, k, v, g, state, start), dict(do=do, dfinal=dfinal), dtype)
    names = ("o", "final", "dq", "dk", "dv", "dstate")
    for name, x, r, b in zip(names, got, refs, bounds):
        assert_close(x, r, b, name)
    again = _grads(ops, q, k, v, g, state, start, do, dfinal)
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # a fixed order of sums
    with torch.no_grad():  # the inference form is the same pass
        o, final = ops.decay_attention(q, k, v, g, state, start)
    assert torch.equal(o, got[0]) and torch.equal(final, got[1])


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_long_axis_with_few_heads(ops, dtype):
    """one env, thousands of steps: whatever splits the axis, the sums are those of the definition"""
    q, k, v, g, state, start, do, dfinal = _case(3001, 1, 2, 32, 24, dtype, 0.0, True, seed=5)
    for st in (None, (torch.rand(3001, 1, generator=_gen(6)) < 0.002).to(DEV)):
        got = _grads(ops, q, k, v, g, state, st, do, dfinal)
        refs, bounds = decay_bounds((q, k, v, g, state, st), dict(do=do, dfinal=dfinal), dtype)
        for name, x, r, b in zip(("o", "final", "dq", "dk", "dv", "dstate"), got, refs, bounds):
            assert_close(x, r, b, name)


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_very_long_axis(ops, dtype):
    """over 32 pieces of the axis, whose states are joined in longer runs"""
    q, k, v, g, state, _, do, dfinal = _case(5003, 1, 2, 17, 32, dtype, 0.0, True, seed=51)
    start = (torch.rand(5003, 1, generator=_gen(52)) < 0.001).to(DEV)
    got = _grads(ops, q, k, v, g, state, start, do, dfinal)
    refs, bounds = decay_bounds((q, k, v, g, state, start), dict(do=do, dfinal=dfinal), dtype)
    for name, x, r, b in zip(("o", "final", "dq", "dk", "dv", "dstate"), got, refs, bounds):
        assert_close(x, r, b, name)


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_many_envs(ops, dtype):
    q, k, v, g, state, start, do, dfinal = _case(5, 700, 3, 32, 32, dtype, 0.2, True, seed=8)
    got = _grads(ops, q, k, v, g, state, start, do, dfinal)
    refs, bounds = decay_bounds((q, k, v, g, state, start), dict(do=do, dfinal=dfinal), dtype)
    for x, r, b in zip(got, refs, bounds):
        assert_close(x, r, b)


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("envs", [7, 120, 173, 300])
def test_many_heads_of_two_widths(ops, envs, dtype):
    """keys and values of different widths, few heads (one launch for all gradients) to many (two), 32 and 64 columns a wave.
    (The bounds count a rounding as half a step relative to the value.  Below 2^-14 float16's steps no longer shrink with the
    value: they are 2^-24 all the way to zero, so the rounding of an answer there is off by up to 2^-25, whatever its size.)"""
    for steps, dk, dv in ((35, 20, 40), (6, 64, 24)):
        q, k, v, g, state, start, do, dfinal = _case(steps, envs, 3, dk, dv, dtype, 0.1, True, seed=envs)
        got = _grads(ops, q, k, v, g, state, start, do, dfinal)
        refs, bounds = decay_bounds((q, k, v, g, state, start), dict(do=do, dfinal=dfinal), dtype)
        for i, (x, r, b) in enumerate(zip(got, refs, bounds)):
            assert_close(x, r, b + (2.0 ** -25 if x.dtype == torch.float16 else 0), (steps, i))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_strides(ops, dtype):
    """slices of one projection, env-major storage, heads expanded from one, uint8 starts of any stride, odd offsets"""
    steps, envs, heads, dk, dv = 37, 3, 2, 32, 64
    q, k, v, g, state, start, do, dfinal = _case(steps, envs, heads, dk, dv, dtype, 0.1, True, seed=2)
    want = _grads(ops, q, k, v, g, state, start, do, dfinal)
    fused = torch.cat([x.flatten(2) for x in (q, k, v)], -1)
    fq, fk, fv = (x.unflatten(-1, (heads, -1)) for x in fused.split([heads * dk, heads * dk, heads * dv], -1))
    shifted = torch.zeros(fused.numel() + 1, dtype=dtype, device=DEV)[1:].view(fused.shape)  # off every vector's alignment
    shifted.copy_(fused)
    sq, sk, sv = (x.unflatten(-1, (heads, -1)) for x in shifted.split([heads * dk, heads * dk, heads * dv], -1))
    env_major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, do)]
    last = [x.transpose(0, 3).contiguous().transpose(0, 3) for x in (q, k, v, do)]
    wide = torch.zeros(envs, 2 * steps, dtype=torch.uint8, device=DEV)
    wide[:, ::2] = 255 * start.t().to(torch.uint8)
    for a in ((fq, fk, fv, g, state, start, do), (sq, sk, sv, g, state, start, do), (*env_major[:3], g, state, start, env_major[3]),
              (*last[:3], g, state, start, last[3]), (q, k, v, g, state.transpose(0, 1).contiguous().transpose(0, 1), wide[:, ::2].t(), do)):
        for x, y in zip(_grads(ops, *a, dfinal), want):
            assert torch.equal(x.contiguous(), y)
    # one key and value head for all: the gradient of the shared head is the sum over those that use it
    k1, v1 = k[:, :, :1].detach().requires_grad_(), v[:, :, :1].detach().requires_grad_()
    o, final = ops.decay_attention(q, k1.expand_as(q), v1.expand(steps, envs, heads, dv), g, state, start)
    got = torch.autograd.grad((o, final), (k1, v1), (do, dfinal))
    full = _grads(ops, q, k[:, :, :1].expand_as(k).contiguous(), v[:, :, :1].expand_as(v).contiguous(), g, state, start, do, dfinal)
    for x, y in zip(got, (full[3], full[4])):
        assert torch.equal(x, y.sum(2, keepdim=True))
    # a gradient expanded from one number, as o.sum() gives it
    leaf = q.detach().requires_grad_()
    (ones,) = torch.autograd.grad(ops.decay_attention(leaf, k, v, g, state, start)[0].sum(), leaf)
    full = _grads(ops, q, k, v, g, state, start, torch.ones_like(do), torch.zeros_like(dfinal))
    assert torch.equal(ones, full[2])


def test_gradient_is_the_difference(ops):
    """o and the final state are linear in each input: a central difference is the derivative"""
    q, k, v, g, state, start, do, dfinal = _case(70, 2, 2, 24, 40, torch.float32, 0.05, True, seed=11)
    got = _grads(ops, q, k, v, g, state, start, do, dfinal)
    args = [q, k, v, state]
    for i, grad in enumerate(got[2:]):
        d = torch.randn(args[i].shape, generator=_gen(i)).to(DEV)
        ends = []
        for sign in (1, -1):
            a = [x + sign * d if j == i else x for j, x in enumerate(args)]
            o, final = ops.decay_attention(a[0], a[1], a[2], g, a[3], start)
            ends.append((o.double() * do).sum() + (final.double() * dfinal).sum())
        slope, want = (ends[0] - ends[1]) / 2, (grad.double() * d).sum()
        # every one of the N summed values has a rounding error of about 1e-6 of its own size: sqrt(N) of them add up
        size = grad.double().norm() * d.double().norm()
        assert abs(slope - want) <= 1e-5 * size, (i, float(slope), float(want))


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_an_episode_does_not_see_another(ops, dtype):
    """infinities and NaN in the carried state and in an episode stay there, forwards and backwards, also where both episodes
    share a tile; an episode's results are those of the episode alone.  (A chunk that holds such a value is cut otherwise than one
    that does not, so the sums' order differs: each is within its bound of the definition.)"""
    steps, envs, heads, dk, dv = 80, 2, 2, 32, 48
    q, k, v, g, state, _, do, dfinal = _case(steps, envs, heads, dk, dv, dtype, 0.0, True, seed=3)
    for starts in ((0, 20, 41), (0, 20, 21, 30, 38, 41, 44), (0, 20, 33, 41)):
        start = torch.zeros(steps, envs, dtype=torch.bool, device=DEV)
        start[list(starts)] = True
        refs, bounds = decay_bounds((q, k, v, g, state, start), dict(do=do, dfinal=dfinal), dtype)
        for which in range(5):  # in one of q, k, v, do, or in all of them
            bad = [x.clone() for x in (q, k, v, do)]
            for x in bad if which == 4 else bad[which:which + 1]:
                x[20:41:3] = float("nan")
                x[21:41:3] = float("inf")
            got = _grads(ops, *bad[:3], g, torch.full_like(state, float("nan")), start, bad[3], dfinal)
            for i in (0, 2, 3, 4):
                for a, b in ((0, 20), (41, 80)):
                    assert_close(got[i][a:b], refs[i][a:b], bounds[i][a:b], (starts, which, i, a))
            assert_close(got[1], refs[1], bounds[1], (starts, which))
            assert torch.equal(got[5], torch.zeros_like(got[5]))
            if which == 4:
                assert torch.isnan(got[0][40].float()).any()
        clean = _grads(ops, q, k, v, g, state, start, do, dfinal)
        alone = _grads(ops, q[44:], k[44:], v[44:], g, None, None, do[44:], dfinal) if 44 in starts else \
            _grads(ops, q[41:], k[41:], v[41:], g, None, None, do[41:], dfinal)
        n = 80 - alone[0].shape[0]
        for i, (x, y) in enumerate(zip([clean[0][n:], clean[1], *(clean[j][n:] for j in (2, 3, 4))], alone)):
            b = bounds[i] if i == 1 else bounds[i][n:]
            assert ((x.double().cpu() - y.double().cpu()).abs() <= 2 * b).all()


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_a_step_does_not_see_a_later_one(ops, dtype):
    """an infinity or NaN in the middle of an episode: every answer before it is as without it, and so is the gradient of every
    step after it with respect to what does not reach it"""
    steps, at = 75, 44
    q, k, v, g, state, _, do, dfinal = _case(steps, 2, 2, 32, 48, dtype, 0.0, True, seed=21)
    refs, bounds = decay_bounds((q, k, v, g, state), dict(do=do, dfinal=dfinal), dtype)
    for x, value in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (v, float("-inf"))):
        keep = x[at].clone()
        x[at] = value
        got = _grads(ops, q, k, v, g, state, None, do, dfinal)
        x[at] = keep
        assert_close(got[0][:at], refs[0][:at], bounds[0][:at], "o")
        assert_close(got[2][:at], refs[2][:at], bounds[2][:at], "dq")
        assert not torch.isfinite(got[0][at].float()).all()
    keep = do[at].clone()
    do[at] = float("nan")  # reaches the gradients of the steps up to it only
    got = _grads(ops, q, k, v, g, state, None, do, dfinal)
    do[at] = keep
    for i in (3, 4):
        assert_close(got[i][at + 1:], refs[i][at + 1:], bounds[i][at + 1:], i)
        assert torch.isnan(got[i][at].float()).any()


@pytest.mark.parametrize("dtype", ALL, ids=str)
def test_decays_at_their_ends(ops, dtype):
    """no decay at all, at once (-inf), and some so strong that their powers underflow"""
    q, k, v, _, state, start, do, dfinal = _case(50, 2, 4, 16, 16, dtype, 0.05, True, seed=4)
    g = torch.tensor([0.0, float("-inf"), -60.0, -9.0], device=DEV)
    for scale in (None, 1e-4, 30.0):  # (float16 results below its smallest number are zero: half of it is allowed beside the bound)
        got = _grads(ops, q, k, v, g, state, start, do, dfinal, scale=scale)
        refs, bounds = decay_bounds((q, k, v, g, state, start), dict(do=do, dfinal=dfinal, scale=scale), dtype)
        for i, (x, r, b) in enumerate(zip(got, refs, bounds)):
            assert_close(x, r, b + (2.0 ** -25 if dtype == torch.float16 and x.dtype == dtype else 1e-30), (scale, i))
        # a head that forgets at once sees its own token
        own = (16 ** -0.5 if scale is None else scale) * (q[:, :, 1].double() * k[:, :, 1].double()).sum(-1, keepdim=True) * v[:, :, 1].double()
        assert_close(got[0][:, :, 1], own.cpu(), bounds[0][:, :, 1] + 2.0 ** -25)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_small_and_large_values(ops, dtype):
    """16-bit values far from one: products leave float16's range inside, and the state is still as exact as float32's"""
    q, k, v, g, state, start, do, dfinal = _case(70, 2, 2, 32, 48, dtype, 0.04, True, seed=31)
    for a, b, c, d in ((300, 200, 1e-3, 1e-4), (1e-3, 1e-4, 1000, 100), (1e-4, 3000, 3, 1e-4)):
        args = [(x.float() * f).to(dtype) for x, f in ((q, a), (k, b), (v, c))]
        dd = (do.float() * d).to(dtype)
        got = _grads(ops, *args, g, state, start, dd, dfinal)
        refs, bounds = decay_bounds((*args, g, state, start), dict(do=dd, dfinal=dfinal), dtype)
        for i, (x, r, e) in enumerate(zip(got, refs, bounds)):
            most = float(torch.finfo(dtype).max)
            fits = r.abs() < most * 0.99
            e = torch.where(fits, e + (2.0 ** -25 if dtype == torch.float16 and x.dtype == dtype else 0), torch.full_like(e, float("inf")))
            assert_close(torch.where(fits.to(DEV), x, torch.zeros_like(x)), torch.where(fits, r, torch.zeros_like(r)), e, (a, b, c, d, i))


def test_an_infinity_leaves_the_others_their_precision(ops):
    """float16 values are scaled by their largest inside: one that is infinite does not count, or its neighbours would overflow"""
    dtype, col = torch.float16, 5
    q, k, v, g, state, _, do, dfinal = _case(75, 2, 2, 32, 48, dtype, 0.0, True, seed=41)
    other = [j for j in range(48) if j != col]

    def check(q, k, v, state, spoil, o_at, columns):
        refs, bounds = decay_bounds((q, k, v, g, state), {}, dtype)
        x, index = spoil
        x[index] = float("inf")
        with torch.no_grad():
            o, final = ops.decay_attention(q, k, v, g, state)
        assert float(refs[0].abs().max()) < 6e4  # a float16 each
        assert_close(o[o_at][..., columns], refs[0][o_at][..., columns], bounds[0][o_at][..., columns] + 2.0 ** -25, "o")
        if columns is other:
            assert_close(final[..., other], refs[1][..., other], bounds[1][..., other], "state")

    values = v * 1000
    check(q, k, values, state, (values, (20, 0, 0, col)), slice(None), other)  # one column's token
    big = q * 1000
    check(big, k * 1000, v * 3e-4, state * 1e-3, (big, (60, 0, 0, 3)), slice(0, 60), list(range(48)))  # a later query
    before = state * 1e6
    check(q * 1e-4, k, v, before, (before, (0, 0, 2, col)), slice(None), other)  # one element remembered


def test_a_step_in_place_is_known_to_autograd(ops):
    """a gradient that still needs the state that a step overwrote is refused, not computed from another state"""
    q, k, v, g, state, _, do, _ = _case(3, 2, 2, 16, 16, torch.float32, 0.0, True, seed=42)
    q.requires_grad_()
    o, _ = ops.decay_attention(q, k, v, g, state)
    with torch.no_grad():
        ops.decay_attention_step(q[0], k[0], v[0], g, state, state_out=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(do)
    out = torch.empty_like(state, requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        ops.decay_attention_step(k[0], k[0], v[0], g, state, state_out=out)


def test_missing_gradients_and_scale(ops):
    """gradients through o alone, through the state alone, for some inputs only; a scale of one's own; no autograd at all"""
    q, k, v, g, state, start, do, dfinal = _case(40, 2, 2, 32, 32, torch.float32, 0.05, True, seed=7)
    full = _grads(ops, q, k, v, g, state, start, do, dfinal, scale=0.3)
    refs, bounds = decay_bounds((q, k, v, g, state, start), dict(do=do, dfinal=dfinal, scale=0.3), torch.float32)
    for x, r, b in zip(full, refs, bounds):
        assert_close(x, r, b)
    kq = k.detach().requires_grad_()
    o, final = ops.decay_attention(q, kq, v, g, state, start, scale=0.3)
    (a,) = torch.autograd.grad(o, kq, do, retain_graph=True)
    (b,) = torch.autograd.grad(final, kq, dfinal)
    assert torch.allclose(a + b, full[3], rtol=1e-4, atol=1e-4)
    s = state.detach().requires_grad_()
    o, final = ops.decay_attention(q, k, v, g, s, start, scale=0.3)
    (d,) = torch.autograd.grad((o, final), s, (do, dfinal))
    assert torch.equal(d, full[5])


def test_gradients_of_gradients_are_refused(ops):
    q, k, v, g, *_ = _case(3, 1, 1, 8, 8, torch.float32)
    q.requires_grad_()
    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    for y, leaf in ((ops.decay_attention(q, k, v, g)[0], q), (ops.layer_norm(x), x)):
        with pytest.raises(RuntimeError, match="gradients of gradients"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)


def test_inputs_changed_before_the_backward_pass_are_noticed(ops):
    q, k, v, g, *_ = _case(3, 1, 1, 8, 8, torch.float32)
    q.requires_grad_()
    o, _ = ops.decay_attention(q, k, v, g)
    k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_zero_lengths(ops):
    q, k, v, g, state, _, _, _ = _case(3, 2, 2, 8, 8, torch.float32, 0.0, True)
    o, final = ops.decay_attention(q[:0], k[:0], v[:0], g, state)
    assert o.shape == (0, 2, 2, 8) and torch.equal(final, state) and final.data_ptr() != state.data_ptr()
    o, final = ops.decay_attention(q[:0], k[:0], v[:0], g)
    assert not final.any()
    e = q[:, :0].detach().requires_grad_()
    o, final = ops.decay_attention(e, k[:, :0], v[:, :0], g)
    assert o.shape == (3, 0, 2, 8) and final.shape == (0, 2, 8, 8)
    (o.sum() + final.sum()).backward()
    assert e.grad.shape == e.shape
    o, s = ops.decay_attention_step(q[0, :0], k[0, :0], v[0, :0], g, state[:0])
    assert o.shape == (0, 2, 8) and s.shape == (0, 2, 8, 8)
    x = torch.zeros(0, 5, device=DEV, requires_grad=True)
    w = torch.ones(5, device=DEV, requires_grad=True)
    y = ops.layer_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 5) and not w.grad.any()


# ---- one token ----

@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (1, 4, 32, 32), (5, 3, 48, 80), (130, 2, 64, 64), (3, 2, 128, 128), (7, 1, 33, 17),
                                  (2, 3, 17, 100), (1000, 2, 16, 8)], ids=lambda s: "x".join(map(str, s)))
def test_decay_step(ops, size, dtype):
    envs, heads, dk, dv = size
    q, k, v, g, state, start, _, _ = _case(1, envs, heads, dk, dv, dtype, 0.3, True, seed=envs)
    state[start[0]] = float("nan")  # an episode that starts does not read what was there
    refs, bounds = decay_bounds((q, k, v, g, state, start), {}, dtype)
    before = state.clone()
    o, new = ops.decay_attention_step(q[0], k[0], v[0], g, state, start[0])
    assert torch.equal(torch.nan_to_num(state), torch.nan_to_num(before)) and new.data_ptr() != state.data_ptr()
    assert_close(o, refs[0][0], bounds[0][0], "o")
    assert_close(new, refs[1], bounds[1], "state")
    o2, new2 = ops.decay_attention_step(q[0], k[0], v[0], g, state, start[0].to(torch.uint8), state_out=state)
    assert new2 is state and torch.equal(o2, o) and torch.equal(state, new)


def test_steps_are_the_sequence(ops):
    """a rollout token by token and the recorded rollout at once: the same answers and the same state"""
    for dtype in ALL:
        q, k, v, g, state, start, _, _ = _case(45, 6, 2, 32, 48, dtype, 0.1, True, seed=9)
        o, final = ops.decay_attention(q, k, v, g, state, start)
        s, outs = state.clone(), []
        for t in range(45):
            y, s = ops.decay_attention_step(q[t], k[t], v[t], g, s, start[t], state_out=s)
            outs.append(y)
        _, bounds = decay_bounds((q, k, v, g, state, start), {}, dtype)
        for x, y, b in zip((o, final), (torch.stack(outs), s), bounds):
            assert ((x.double().cpu() - y.double().cpu()).abs() <= 2 * b).all()


def test_step_strides(ops):
    q, k, v, g, state, start, _, _ = _case(1, 9, 2, 32, 32, torch.bfloat16, 0.3, True, seed=1)
    want = ops.decay_attention_step(q[0], k[0], v[0], g, state, start[0])
    fused = torch.cat([torch.zeros_like(q[0, :, :, :1]).flatten(1)] + [x[0].flatten(1) for x in (q, k, v)], -1)
    fq, fk, fv = (fused[:, 2 + 64 * i:66 + 64 * i].unflatten(-1, (2, 32)) for i in range(3))
    got = ops.decay_attention_step(fq, fk, fv, g, state, torch.stack([start[0], ~start[0]], 1)[:, 0])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    moved = torch.zeros(state.numel() + 1, device=DEV)[1:].view(state.shape)  # a state off 16-byte alignment
    moved.copy_(state)
    got = ops.decay_attention_step(q[0], k[0], v[0], g, moved, start[0], state_out=moved)
    assert torch.equal(moved, want[1])  # each element is one product and one sum, in any layout
    refs, bounds = decay_bounds((q, k, v, g, state, start), {}, torch.bfloat16)
    assert_close(got[0], refs[0][0], bounds[0][0])  # o's sum runs in another order there: each order is within its bound


# ---- layer norm ----

NORMS = [((1, 1), True), ((3, 2), True), ((1, 7), False), ((5, 17), True), ((300, 17), True), ((64, 9), True), ((2049, 6), True),
         ((33, 64), True), ((100, 256), True), ((7, 255), True), ((9, 1000), True), ((4, 1024), True), ((5, 2500), True),
         ((3, 5000), True), ((2, 8192), True), ((2, 9001), False), ((6, 5, 4, 32), True), ((1500, 128), False)]


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("shape,affine", NORMS, ids=lambda s: str(s))
def test_layer_norm(ops, shape, affine, dtype):
    gen = _gen(len(shape) + shape[0])
    x = (1.5 * torch.randn(*shape, generator=gen) + torch.randn(*shape[:-1], 1, generator=gen)).to(dtype).to(DEV)
    dy = torch.randn(*shape, generator=gen).to(dtype).to(DEV)
    for pdtype in sorted({dtype, torch.float32}, key=str) if affine else (None,):
        w = (1 + 0.1 * torch.randn(shape[-1], generator=gen)).to(pdtype).to(DEV).requires_grad_() if affine else None
        b = (0.1 * torch.randn(shape[-1], generator=gen)).to(pdtype).to(DEV).requires_grad_() if affine else None
        leaf = x.detach().requires_grad_()
        y = ops.layer_norm(leaf, w, b, eps=1e-5)
        leaves = (leaf, w, b) if affine else (leaf,)
        got = (y, *torch.autograd.grad(y, leaves, dy))
        refs, bounds = norm_bounds(x, w, b, 1e-5, dy)
        for name, a, r, e in zip(("y", "dx", "dw", "db"), got, refs, bounds):
            assert_close(a, r, e, name)
        y2 = ops.layer_norm(leaf, w, b, eps=1e-5)
        for a, c in zip(got, (y2, *torch.autograd.grad(y2, leaves, dy))):
            assert torch.equal(a, c)  # a fixed order of sums
        with torch.no_grad():
            assert torch.equal(ops.layer_norm(x, w, b), y)


def test_layer_norm_many_wide_rows(ops):
    """rows that no workgroup holds at once, more of them than workgroups"""
    x = (torch.randn(700, 8195, generator=_gen(71)) + 0.5).to(DEV).requires_grad_()
    dy, w = torch.randn(700, 8195, generator=_gen(72)).to(DEV), torch.full((8195,), 1.25, device=DEV, requires_grad=True)
    y = ops.layer_norm(x, w)
    refs, bounds = norm_bounds(x.detach(), w.detach(), None, 1e-5, dy)
    for name, a, r, e in zip(("y", "dx", "dw"), (y, *torch.autograd.grad(y, (x, w), dy)), refs, bounds):
        assert_close(a, r, e, name)


def test_layer_norm_strides_and_partial_gradients(ops):
    x = torch.randn(6, 5, 24, generator=_gen(0)).to(DEV)
    w, b = torch.randn(24, generator=_gen(1)).to(DEV).requires_grad_(), torch.randn(24, generator=_gen(2)).to(DEV).requires_grad_()
    dy = torch.randn(6, 5, 24, generator=_gen(3)).to(DEV)
    want = ops.layer_norm(x, w, b)
    grads = torch.autograd.grad(want, (w, b), dy)
    pad = torch.zeros(6, 5, 31, device=DEV)
    pad[..., 3:27] = x
    # rows off 16-byte alignment are summed in another order: each of the two sums is within its bound of the definition
    refs, bounds = norm_bounds(x, w, b, 1e-5, dy)
    off = ops.layer_norm(pad[..., 3:27], w, b)
    for a, r, e in zip((off, *torch.autograd.grad(off, (w, b), dy)), (refs[0], *refs[2:]), (bounds[0], *bounds[2:])):
        assert_close(a, r, e)
    pad = torch.zeros(6, 5, 32, device=DEV)
    pad[..., 4:28] = x
    for v in (pad[..., 4:28], x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(0, 2).contiguous().transpose(0, 2)):
        assert torch.equal(ops.layer_norm(v, w, b), want)
        got = torch.autograd.grad(ops.layer_norm(v, w, b), (w, b), dy.transpose(0, 1).contiguous().transpose(0, 1))
        assert all(torch.equal(a, c) for a, c in zip(got, grads))
    row = torch.randn(24, generator=_gen(4)).to(DEV)
    assert torch.equal(ops.layer_norm(row.expand(4, 24), w, b), ops.layer_norm(row.expand(4, 24).contiguous(), w, b))
    assert torch.equal(ops.layer_norm(row), ops.layer_norm(row[None])[0])
    (only_b,) = torch.autograd.grad(ops.layer_norm(x, None, b).sum(), (b,))
    assert torch.equal(only_b, torch.full_like(b, 30.0))
    (only_w,) = torch.autograd.grad(ops.layer_norm(x, w), (w,), dy)
    assert torch.equal(only_w, grads[0])


def test_layer_norm_rows_do_not_meet(ops):
    """a row of NaN or infinities stays one; a constant row gives the bias; large offsets keep their variance"""
    x = torch.randn(9, 300, generator=_gen(5)).to(DEV)
    want = ops.layer_norm(x)
    x[3], x[7, 5] = float("nan"), float("inf")
    got = ops.layer_norm(x)
    keep = [0, 1, 2, 4, 5, 6, 8]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[3]).all() and torch.isnan(got[7]).all()
    b = torch.randn(300, generator=_gen(6)).to(DEV)
    assert torch.equal(ops.layer_norm(torch.full((2, 300), 0.25, device=DEV), None, b), b.expand(2, 300))
    far = 1000.0 + torch.randn(4, 300, generator=_gen(7))
    refs, bounds = norm_bounds(far, None, None, 1e-5)
    assert_close(ops.layer_norm(far.to(DEV)), refs[0], bounds[0])
    assert float(bounds[0].max()) < 0.5  # the bound itself still says something


# ---- streams, graphs, buffers ----

def test_another_stream_and_its_gradients(ops):
    q, k, v, g, state, start, do, dfinal = _case(64, 4, 2, 32, 32, torch.bfloat16, 0.05, True, seed=12)
    want = _grads(ops, q, k, v, g, state, start, do, dfinal)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = [x.clone() for x in (q, k, v)]
        busy = torch.randn(2048, 2048, device=DEV)
        for _ in range(4):
            busy = busy @ busy * 1e-2
        late = [x + 0 * busy[0, 0].to(x.dtype).nan_to_num() for x in late]
        got = _grads(ops, *late, g, state, start, do, dfinal)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_rollout_step_and_training_step(ops):
    """the token step and a training pass in two graphs, replayed in turn with eager work between, each replay checked"""
    q, k, v, g, state, start, do, dfinal = _case(70, 3, 2, 32, 64, torch.bfloat16, 0.05, True, seed=13)
    x = torch.randn(50, 64, generator=_gen(14)).to(DEV)
    w, b = torch.ones(64, device=DEV, requires_grad=True), torch.zeros(64, device=DEV, requires_grad=True)

    def train():
        y = ops.layer_norm(x, w, b)
        return [*_grads(ops, q, k, v, g, state, start, do, dfinal), y, *torch.autograd.grad(y, (w, b), x)]

    memory = state.clone()

    def step():
        return ops.decay_attention_step(q[0], k[0], v[0], g, memory, start[0], state_out=memory)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(), step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph1, graph2, graph3 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph1):
        out = train()
    with torch.cuda.graph(graph2):
        y = step()
    with torch.cuda.graph(graph3):
        out3 = train()
    memory.copy_(state)
    eager = state.clone()
    for i in range(4):
        for t in (q, k, v, x):
            t.copy_(torch.randn(t.shape, generator=_gen(20 + i)).to(t.dtype))
        torch.cuda.synchronize()
        graph1.replay(), graph2.replay(), graph3.replay()
        want = train()
        assert all(torch.equal(a, c) for a, c in zip(out, want)) and all(torch.equal(a, c) for a, c in zip(out3, want))
        y2, eager = ops.decay_attention_step(q[0], k[0], v[0], g, eager, start[0])
        assert torch.equal(y, y2) and torch.equal(memory, eager)
        torch.cuda.synchronize()


def test_captured_odd_widths_and_a_long_axis(ops):
    """two captured passes that need copies of their inputs and the axis cut up, each with its own workspace, replayed in turn"""
    cases = [_case(steps, 1, 2, 17, 33, torch.float16, 0.01, True, seed=steps) for steps in (700, 1500)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cases:
            _grads(ops, *c)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in cases], []
    for graph, c in zip(graphs, cases):
        with torch.cuda.graph(graph):
            outs.append(_grads(ops, *c))
    for i in range(3):
        for c in cases:
            for t in c[:3]:
                t.copy_(torch.randn(t.shape, generator=_gen(60 + i)).to(t.dtype))
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        for out, c in zip(outs, cases):
            assert all(torch.equal(a, b) for a, b in zip(out, _grads(ops, *c)))
        torch.cuda.synchronize()


def test_nothing_is_written_beyond_the_outputs(ops):
    """the C entries on buffers inside larger ones: what lies before and behind stays as it was"""
    from urgym_amd.ops import _native
    L = _native.lib()
    codes = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}
    for dtype in ALL:
        q, k, v, g, state, start, do, dfinal = _case(35, 3, 2, 24, 40, dtype, 0.1, True, seed=15)
        s = _native.Seq(codes[dtype], 2, 24, 40, 35, 3, q.data_ptr(), k.data_ptr(), v.data_ptr())
        s.q_stride[:], s.k_stride[:], s.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
        s.log_decay, s.start, s.start_stride[:], s.state, s.scale = g.data_ptr(), start.data_ptr(), start.stride(), state.data_ptr(), 0.2

        def framed(n, dt):
            return torch.full((n + 512,), 7.0, dtype=dt, device=DEV)
        sizes = [(35 * 3 * 2 * 40, dtype), (3 * 2 * 24 * 40, torch.float32), (35 * 3 * 2 * 24, dtype), (35 * 3 * 2 * 24, dtype),
                 (35 * 3 * 2 * 40, dtype), (3 * 2 * 24 * 40, torch.float32)]
        bufs = [framed(*z) for z in sizes]
        stride = (ctypes.c_int64 * 3)(*do.stride()[:3])
        n = [L.urgym_ops_decay_workspace(ctypes.byref(s)), L.urgym_ops_decay_backward_workspace(ctypes.byref(s), do.data_ptr(), stride)]
        ws = [framed(x, torch.float32) for x in n]
        at = [x[256:].data_ptr() for x in bufs]
        wat = [x[256:].data_ptr() if m else None for x, m in zip(ws, n)]
        stream = torch.cuda.current_stream().cuda_stream
        assert L.urgym_ops_decay(ctypes.byref(s), at[0], at[1], wat[0], stream) == 0
        assert L.urgym_ops_decay_backward(ctypes.byref(s), do.data_ptr(), stride, dfinal.data_ptr(), *at[2:], wat[1], stream) == 0
        want = _grads(ops, q, k, v, g, state, start, do, dfinal, scale=0.2)
        for buf, y in zip(bufs, want):
            assert torch.equal(buf[256:-256], y.flatten()) and (buf[:256] == 7).all() and (buf[-256:] == 7).all()
        for buf in ws:
            assert (buf[:256] == 7).all() and (buf[-256:] == 7).all()
        rows, width = 37, 19
        x = torch.randn(rows, width, generator=_gen(1)).to(dtype).to(DEV)
        w = torch.ones(width, device=DEV)
        y, stats, dx, dw, db = framed(rows * width, dtype), framed(2 * rows, torch.float32), framed(rows * width, dtype), \
            framed(width, torch.float32), framed(width, torch.float32)
        ws = framed(L.urgym_ops_layer_norm_workspace(rows, width), torch.float32)
        code, p = codes[dtype], lambda t, i=0: t[256 + i:].data_ptr()  # noqa: E731
        assert L.urgym_ops_layer_norm(code, 0, rows, width, x.data_ptr(), width, w.data_ptr(), None, 1e-5, p(y), p(stats),
                                      p(stats, rows), stream) == 0
        assert L.urgym_ops_layer_norm_backward(code, 0, rows, width, x.data_ptr(), width, x.data_ptr(), width, w.data_ptr(),
                                               p(stats), p(stats, rows), p(dx), p(dw), p(db), p(ws), stream) == 0
        for buf in (y, stats, dx, dw, db, ws):
            assert (buf[:256] == 7).all() and (buf[-256:] == 7).all()


def test_far_offsets(ops):
    """strides whose byte offsets pass 32 bits: the last step's token lies beyond 4 GiB"""
    base = torch.zeros(5 * (1 << 29) + 4096, dtype=torch.bfloat16, device=DEV)
    step = 1 << 29
    views = [base[i * 256:].as_strided((5, 2, 2, 32), (step, 64, 32, 1)) for i in range(4)]
    q, k, v, g, state, start, do, dfinal = _case(5, 2, 2, 32, 32, torch.bfloat16, 0.0, True, seed=16)
    for far, near in zip(views, (q, k, v, do)):
        far.copy_(near)
    for a, b in zip(_grads(ops, *views[:3], g, state, start, views[3], dfinal), _grads(ops, q, k, v, g, state, start, do, dfinal)):
        assert torch.equal(a, b)
    rows = base.as_strided((5, 64), (step, 1))
    assert torch.equal(ops.layer_norm(rows), ops.layer_norm(rows.contiguous()))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="one GPU")
def test_another_device_than_the_current_one(ops):
    x = torch.randn(5, 33, generator=_gen(0))
    assert torch.equal(ops.layer_norm(x.to("cuda:1")).cpu(), ops.layer_norm(x.to("cuda:0")).cpu())


def test_devices_must_agree(ops):
    x = torch.zeros(3, 4, device=DEV)
    with pytest.raises(ValueError):
        ops.layer_norm(x, torch.ones(4))
    q = torch.zeros(2, 1, 1, 4, device=DEV)
    with pytest.raises(ValueError):
        ops.decay_attention(q, q, q, torch.zeros(1))
    with pytest.raises(ValueError):
        ops.decay_attention(q, q, q, torch.zeros(1, device=DEV), start=torch.zeros(2, 1, dtype=torch.bool))
