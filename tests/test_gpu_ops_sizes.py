"""The policy operators at the sizes that large launches take: 64 columns of the state a wave (heads of 33 to 64, many of them), and the
widest rows that the layer norm's groups hold -- against the definitions in 64 bits (tests/ops_reference.py)."""
import pytest
import torch

from ops_reference import assert_close, decay_bounds, norm_bounds

pytestmark = pytest.mark.gpu
DEV = "cuda"
ALL = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("o", "final", "dq", "dk", "dv", "dstate")


@pytest.fixture(scope="module")
def ops(built):
    from urgym_amd import ops
    return ops


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("steps,envs,heads,dk,dv", [(35, 345, 3, 64, 64), (35, 345, 3, 48, 40), (35, 345, 3, 64, 128), (97, 1031, 1, 64, 64),
                                                    (150, 130, 8, 64, 64), (18, 257, 4, 33, 61), (66, 520, 2, 128, 64), (130, 340, 3, 40, 64)])
def test_many_heads_of_64(ops, steps, envs, heads, dk, dv, dtype):
    """(every env is run; the definition is computed for some of them)"""
    gen = torch.Generator(device=DEV).manual_seed(steps + dk)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    q, k, v, do = (r(steps, envs, heads, d).to(dtype) for d in (dk, dk, dv, dv))
    state, dfinal = 3 * r(envs, heads, dk, dv), r(envs, heads, dk, dv)
    decay = torch.log1p(-1.0 / torch.logspace(0.5, 6, heads, base=2.0)).to(DEV) if heads > 1 else torch.tensor([-0.05], device=DEV)
    start = torch.rand(steps, envs, generator=gen, device=DEV) < 0.04
    some = torch.tensor([0, 1, envs // 2, envs - 2, envs - 1], device=DEV)
    for carry, starts in ((state, start), (None, None)):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([state.detach().requires_grad_()] if carry is not None else [])
        o, final = ops.decay_attention(*leaves[:3], decay, leaves[3] if carry is not None else None, starts)
        got = [o, final, *torch.autograd.grad((o, final), leaves, (do, dfinal))]
        args = [x[:, some] for x in (q, k, v)] + [decay, None if carry is None else carry[some], None if starts is None else starts[:, some]]
        refs, bounds = decay_bounds(args, dict(do=do[:, some], dfinal=dfinal[some]), dtype)
        for name, x, ref, b in zip(NAMES, got, refs, bounds):
            assert torch.isfinite(x.float()).all(), name
            y = x[some] if name in ("final", "dstate") else x[:, some]
            assert_close(y, ref, b + (2.0 ** -25 if y.dtype == torch.float16 else 0), (name, carry is None))
        with torch.no_grad():
            o2, final2 = ops.decay_attention(q, k, v, decay, carry, starts)
        assert torch.equal(o2, o) and torch.equal(final2, final)


WIDE = [(5, 4095), (5, 8191), (3, 8192), (300, 8184), (3, 12288), (4, 16384), (3, 16392), (3, 32768), (260, 20000), (2, 32776), (600, 4104)]


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("rows,width", WIDE)
def test_layer_norm_of_wide_rows(ops, rows, width, dtype):
    gen = torch.Generator().manual_seed(width)
    x = (1.5 * torch.randn(rows, width, generator=gen) + torch.randn(rows, 1, generator=gen)).to(dtype).to(DEV)
    dy = torch.randn(rows, width, generator=gen).to(dtype).to(DEV)
    for pdtype in sorted({dtype, torch.float32}, key=str):
        w = (1 + 0.1 * torch.randn(width, generator=gen)).to(pdtype).to(DEV).requires_grad_()
        b = (0.1 * torch.randn(width, generator=gen)).to(pdtype).to(DEV).requires_grad_()
        leaf = x.detach().requires_grad_()
        y = ops.layer_norm(leaf, w, b)
        refs, bounds = norm_bounds(x, w, b, 1e-5, dy)
        for name, a, r, e in zip(("y", "dx", "dw", "db"), (y, *torch.autograd.grad(y, (leaf, w, b), dy)), refs, bounds):
            assert_close(a, r, e + (2.0 ** -25 if a.dtype == torch.float16 else 0), (name, pdtype))
        y = ops.layer_norm(x, w, b)
        (dw,) = torch.autograd.grad(y, (w,), dy)  # without x's gradient
        assert_close(dw, refs[2], bounds[2] + (2.0 ** -25 if dw.dtype == torch.float16 else 0))


@pytest.mark.parametrize("dtype", ALL, ids=str)
@pytest.mark.parametrize("width", [60, 512, 516, 600, 1004, 1200, 1537, 2048, 2052, 4100])
def test_layer_norm_workspace_is_enough(ops, width, dtype):
    """the C entry says how much, whatever the type and the rows' alignment: nothing is written behind it, and the sums are right"""
    from urgym_amd.ops import _native
    L = _native.lib()
    code = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}[dtype]
    rows, stream = 1100, torch.cuda.current_stream().cuda_stream
    gen = torch.Generator().manual_seed(width)
    n = L.urgym_ops_layer_norm_workspace(rows, width)
    for pad in (0, 1):  # rows that start anywhere: single elements
        x = torch.randn(rows, width + pad, generator=gen).to(dtype).to(DEV)[:, pad:]
        dy = torch.randn(rows, width, generator=gen).to(dtype).to(DEV)
        w = torch.ones(width, device=DEV)
        y, dx = torch.empty_like(dy), torch.empty_like(dy)
        stats, dw, db = torch.empty(2, rows, device=DEV), torch.empty(width, device=DEV), torch.empty(width, device=DEV)
        ws = torch.full((n + 4096,), 7.0, device=DEV)
        assert L.urgym_ops_layer_norm(code, 0, rows, width, x.data_ptr(), x.stride(0), w.data_ptr(), None, 1e-5, y.data_ptr(), stats[0].data_ptr(),
                                      stats[1].data_ptr(), stream) == 0
        assert L.urgym_ops_layer_norm_backward(code, 0, rows, width, dy.data_ptr(), width, x.data_ptr(), x.stride(0), w.data_ptr(),
                                               stats[0].data_ptr(), stats[1].data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                               ws.data_ptr(), stream) == 0
        assert (ws[n:] == 7).all()
        refs, bounds = norm_bounds(x, w, None, 1e-5, dy)
        for name, a, r, e in zip(("y", "dx", "dw", "db"), (y, dx, dw, db), refs, bounds):
            assert_close(a, r, e + (2.0 ** -25 if a.dtype == torch.float16 else 0), (name, pad))


@pytest.mark.parametrize("dtype,steps,envs,dk,dv", [(torch.bfloat16, 31, 300001, 64, 8), (torch.float16, 32, 300001, 8, 128),
                                                    (torch.float32, 15, 300001, 64, 8), (torch.float32, 16, 300001, 8, 65),
                                                    (torch.bfloat16, 63, 300001, 65, 9)], ids=str)
def test_steps_that_lie_far_apart(ops, dtype, steps, envs, dk, dv):
    """batches whose steps take 150 MB and more: a chunk of them lies over more than 4 GiB"""
    heads = 4
    gen = torch.Generator(device=DEV).manual_seed(dk)
    q, k, v, do = (torch.empty(steps, envs, heads, d, dtype=dtype, device=DEV).normal_(generator=gen) for d in (dk, dk, dv, dv))
    dfinal = torch.empty(envs, heads, dk, dv, device=DEV).normal_(generator=gen)
    decay = torch.tensor([-0.5, -0.2, -0.05, -0.01], device=DEV)
    start = torch.rand(steps, envs, generator=gen, device=DEV) < 0.03
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o, final = ops.decay_attention(*leaves, decay, None, start)
    got = [o, final, *torch.autograd.grad((o, final), leaves, (do, dfinal))]
    some = torch.tensor([0, 1, envs // 2, envs - 1], device=DEV)
    refs, bounds = decay_bounds([x.detach()[:, some] for x in (q, k, v)] + [decay, None, start[:, some]], dict(do=do[:, some], dfinal=dfinal[some]), dtype)
    for name, x, ref, b in zip(NAMES, got, refs, bounds):
        y = x.detach()
        y = y[some] if name == "final" else y[:, some]
        assert_close(y, ref, b + (2.0 ** -25 if y.dtype == torch.float16 else 0), name)
