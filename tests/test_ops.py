"""The policy operators without a GPU: the library exports what include/urgym_ops.h declares, the arguments are checked before
anything is enqueued, and the reference that the GPU tests compare with is itself checked against autograd."""
import ctypes
import os
import re

import pytest
import torch

from ops_reference import decay_reference, norm_reference
from urgym_amd import ops
from urgym_amd.ops import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _heads(steps=3, envs=2, heads=2, dk=4, dv=6, dtype=torch.float32):
    return (torch.zeros(steps, envs, heads, dk, dtype=dtype), torch.zeros(steps, envs, heads, dk, dtype=dtype),
            torch.zeros(steps, envs, heads, dv, dtype=dtype), torch.zeros(heads))


def test_header_binding_and_library_agree(built):
    txt = open(os.path.join(ROOT, "include", "urgym_ops.h")).read()
    declared = sorted(set(re.findall(r"\b(urgym_ops_[a-z_]+)\s*\(", txt)))
    assert sorted(_native.SYMBOLS) == declared
    L = _native.lib()
    for s in declared:
        assert hasattr(L, s), s


def test_no_cpu_fallback(built):
    q, k, v, g = _heads()
    for call in (lambda: ops.layer_norm(torch.zeros(3, 4)), lambda: ops.decay_attention(q, k, v, g),
                 lambda: ops.decay_attention_step(q[0], k[0], v[0], g, torch.zeros(2, 2, 4, 6))):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()


def test_layer_norm_refusals(built):
    x = torch.zeros(3, 4)
    for bad in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x, torch.zeros(4, dtype=torch.bfloat16)),
                lambda: ops.layer_norm([1.0]), lambda: ops.layer_norm(x.half(), torch.zeros(4), torch.zeros(4).half())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: ops.layer_norm(x, torch.zeros(3)), lambda: ops.layer_norm(x, None, torch.zeros(1, 4)),
                lambda: ops.layer_norm(torch.zeros(3, 0)), lambda: ops.layer_norm(torch.zeros(())),
                lambda: ops.layer_norm(x, eps=0.0), lambda: ops.layer_norm(x, eps=float("nan"))):
        with pytest.raises(ValueError):
            bad()


def test_decay_attention_refusals(built):
    q, k, v, g = _heads()
    for bad in (lambda: ops.decay_attention(q.double(), k.double(), v.double(), g),
                lambda: ops.decay_attention(q, k.half(), v, g), lambda: ops.decay_attention(q, k, v, g.double()),
                lambda: ops.decay_attention(q, k, v, g, state=torch.zeros(2, 2, 4, 6).half()),
                lambda: ops.decay_attention(q, k, v, g, start=torch.zeros(3, 2)), lambda: ops.decay_attention(q, k, None, g)):
        with pytest.raises(TypeError):
            bad()
    wide = torch.zeros(3, 2, 2, 129)
    for bad in (lambda: ops.decay_attention(q[0], k[0], v[0], g), lambda: ops.decay_attention(q, k[:2], v, g),
                lambda: ops.decay_attention(q, k, v[:, :1], g), lambda: ops.decay_attention(wide, wide, v, g),
                lambda: ops.decay_attention(q, k, wide, g), lambda: ops.decay_attention(q[..., :0], k[..., :0], v, g),
                lambda: ops.decay_attention(q[:, :, :0], k[:, :, :0], v[:, :, :0], g[:0]),
                lambda: ops.decay_attention(q, k, v, g[:1]), lambda: ops.decay_attention(q, k, v, g.clone().requires_grad_()),
                lambda: ops.decay_attention(q, k, v, g, state=torch.zeros(2, 2, 6, 4)),
                lambda: ops.decay_attention(q, k, v, g, start=torch.zeros(2, 3, dtype=torch.bool))):
        with pytest.raises(ValueError):
            bad()


def test_decay_attention_step_refusals(built):
    q, k, v, g = _heads()
    q, k, v, s = q[0], k[0], v[0], torch.zeros(2, 2, 4, 6)
    big = torch.zeros(2 * 48 * 2 + 8)
    for bad in (lambda: ops.decay_attention_step(q, k, v, g, s[:1]), lambda: ops.decay_attention_step(q, k, v, g, s.transpose(0, 1)),
                lambda: ops.decay_attention_step(q, k, v, g, s, start=torch.zeros(3, dtype=torch.bool)),
                lambda: ops.decay_attention_step(q, k, v, g, s, state_out=s[:1]),
                lambda: ops.decay_attention_step(q, k, v, g, big[:96].view(2, 2, 4, 6), state_out=big[8:104].view(2, 2, 4, 6)),
                lambda: ops.decay_attention_step(q.clone().requires_grad_(), k, v, g, s)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.decay_attention_step(q, k, v, g, None)


def test_library_refuses_bad_sizes_without_a_gpu(built):
    """the C entries check what they are given before they enqueue anything, and say what was wrong"""
    L = _native.lib()
    assert L.urgym_ops_layer_norm(7, 0, 1, 1, None, 1, None, None, 1e-5, None, None, None, None) == -1
    assert b"dtype" in L.urgym_ops_last_error()
    assert L.urgym_ops_layer_norm(0, 0, 1, 0, None, 1, None, None, 1e-5, None, None, None, None) == -1
    assert L.urgym_ops_layer_norm(0, 0, 1, 4, None, 4, None, None, 1e-5, None, None, None, None) == -1
    assert L.urgym_ops_layer_norm_backward(1, 2, 1, 4, *[None] * 1, 4, None, 4, *[None] * 8) == -1
    s = _native.Seq(0, 2, 200, 4, 3, 1)
    assert L.urgym_ops_decay(ctypes.byref(s), None, None, None, None) == -1 and b"200" in L.urgym_ops_last_error()
    s = _native.Seq(0, 2, 4, 4, 0, 1)
    assert L.urgym_ops_decay(ctypes.byref(s), None, None, None, None) == -1
    s = _native.Seq(0, 8, 4, 4, 3, 1 << 20)  # more heads than a launch has room for
    assert L.urgym_ops_decay(ctypes.byref(s), None, None, None, None) == -1 and b"too large" in L.urgym_ops_last_error()
    assert L.urgym_ops_decay_workspace(ctypes.byref(s)) == -1
    s = _native.Seq(0, 2, 4, 4, 3, 1)
    assert L.urgym_ops_decay(ctypes.byref(s), None, None, None, None) == -1 and b"needed" in L.urgym_ops_last_error()
    assert L.urgym_ops_decay_step(0, 1, 1, 4, 4, *[None, 0, 0] * 3, None, None, 0, 1.0, None, None, None, None) == -1


def test_reference_gradients_match_autograd():
    torch.manual_seed(0)
    q, k = (torch.randn(7, 2, 3, 4, dtype=torch.float64, requires_grad=True) for _ in range(2))
    v = torch.randn(7, 2, 3, 5, dtype=torch.float64, requires_grad=True)
    s0 = torch.randn(2, 3, 4, 5, dtype=torch.float64, requires_grad=True)
    g = -torch.rand(3, dtype=torch.float64)
    start = torch.rand(7, 2) < 0.3
    s, o = s0, []
    for t in range(7):
        s = torch.where(start[t][:, None, None, None], torch.zeros_like(s), g.exp()[:, None, None] * s) + k[t][..., None] * v[t][..., None, :]
        o.append(0.7 * (q[t][..., None] * s).sum(-2))
    o = torch.stack(o)
    do, ds = torch.randn_like(o), torch.randn_like(s)
    want = (o, s, *torch.autograd.grad((o, s), (q, k, v, s0), (do, ds)))
    got = decay_reference(q, k, v, g, s0, start, 0.7, do, ds)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
    x, w, b = torch.randn(6, 9, dtype=torch.float64, requires_grad=True), torch.randn(9).double().requires_grad_(), torch.randn(9).double().requires_grad_()
    y = torch.nn.functional.layer_norm(x, (9,), w, b, 1e-5)
    dy = torch.randn_like(y)
    for a, c in zip(norm_reference(x, w, b, 1e-5, dy), (y, *torch.autograd.grad(y, (x, w, b), dy))):
        assert torch.allclose(a, c, rtol=1e-10, atol=1e-12)
