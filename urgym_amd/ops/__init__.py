"""Operators of policies with memory, as HIP kernels (liburgym_ops.so, include/urgym_ops.h).

The tasks observe positions, not velocities, so a policy that is to know how fast the ball rolls has to remember.  These are
the operators such a policy is made of, in the layout of the vector envs: time-major [steps, envs, ...], a state per env,
and the env's done flags as episode starts.

* `decay_attention` -- linear attention with a decay for each head over a recorded rollout, with gradients;
* `decay_attention_step` -- its recurrent form: one token per env, inside a rollout;
* `layer_norm` -- layer norm over the last axis, with gradients.

Tensors are torch tensors on one GPU; every kernel is enqueued on torch's current stream of that GPU and may be captured into a
graph (outputs and workspaces come from torch's allocator, so each captured graph has its own).  When a training step is
captured, no autograd graph of an earlier eager pass over the same parameters may still be alive: torch ties a parameter's
gradient accumulation to the stream of the pass that first used it, and joining that stream inside a capture fails.
Drop the eager outputs first, or capture `torch.autograd.grad`.  Gradients of gradients are not offered.
Errors: ValueError / TypeError for arguments, RuntimeError for what the library reports.  There is no CPU fallback.
"""
import ctypes
import os

import torch

_LIB_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_lib", "liburgym_ops.so")
# C-ABI symbols declared in include/urgym_ops.h
SYMBOLS = ["urgym_ops_last_error", "urgym_ops_layer_norm", "urgym_ops_layer_norm_workspace", "urgym_ops_layer_norm_backward",
           "urgym_ops_decay_workspace", "urgym_ops_decay", "urgym_ops_decay_backward", "urgym_ops_decay_step"]
MAX_HEAD_DIM = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_lib = None


class _Seq(ctypes.Structure):  # urgym_ops_seq
    _fields_ = [("dtype", ctypes.c_int32), ("heads", ctypes.c_int32), ("dk", ctypes.c_int32), ("dv", ctypes.c_int32),
                ("steps", ctypes.c_int64), ("envs", ctypes.c_int64),
                ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("q_stride", ctypes.c_int64 * 3), ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
                ("log_decay", ctypes.c_void_p), ("start", ctypes.c_void_p), ("start_stride", ctypes.c_int64 * 2),
                ("state", ctypes.c_void_p), ("scale", ctypes.c_float)]


def lib():
    """The loaded library; RuntimeError if it is not built."""
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            raise RuntimeError(f"{os.path.basename(_LIB_PATH)} not built ({_LIB_PATH}); run __graft_entry__.build() -- "
                               "no CPU fallback exists")
        L = ctypes.CDLL(_LIB_PATH)
        P, I, Q, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        L.urgym_ops_last_error.restype = ctypes.c_char_p
        L.urgym_ops_layer_norm.argtypes = [I, I, Q, Q, P, Q, P, P, F, P, P, P, P]
        L.urgym_ops_layer_norm_workspace.argtypes = [Q, Q]
        L.urgym_ops_layer_norm_workspace.restype = Q
        L.urgym_ops_layer_norm_backward.argtypes = [I, I, Q, Q, P, Q, P, Q, P, P, P, P, P, P, P, P]
        L.urgym_ops_decay_workspace.argtypes = [ctypes.POINTER(_Seq), I]
        L.urgym_ops_decay_workspace.restype = Q
        L.urgym_ops_decay.argtypes = [ctypes.POINTER(_Seq), P, P, P, P]
        L.urgym_ops_decay_backward.argtypes = [ctypes.POINTER(_Seq), P, Q * 3, P, P, P, P, P, P, P]
        L.urgym_ops_decay_step.argtypes = [I, Q, I, I, I, P, Q, Q, P, Q, Q, P, Q, Q, P, P, Q, F, P, P, P, P]
        _lib = L
    return _lib


def _check(rc):
    if rc:
        raise RuntimeError(_lib.urgym_ops_last_error().decode())


class _on:
    """torch's current stream of x's device, with that device current while a kernel is enqueued"""

    def __init__(self, x):
        self.index = x.device.index
        self.guard = None

    def __enter__(self):
        if torch.cuda.current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _need(name, x, dtypes, device=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, not {type(x).__name__}")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, not {x.dtype}")
    if device is not None and x.device != device:
        raise ValueError(f"{name} is on {x.device}, not on {device}")


def _need_gpu(x):
    if x.device.type != "cuda":
        raise ValueError(f"the operators run on the GPU, the tensors are on {x.device}; no CPU fallback exists")


def _rows(x):
    """x with its last axis contiguous (a copy only if it is not)"""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _ptr(x):
    return None if x is None else x.data_ptr()


# ---- layer norm ----

def _matrix(x, width):
    """x as [rows, width] and its row stride (a view where its leading axes allow one)"""
    m = _rows(x).reshape(-1, width)
    if m.stride(-1) != 1 and width > 1:
        m = m.contiguous()
    return m, m.stride(0) if m.shape[0] > 1 else width


def _norm_forward(x, weight, bias, eps, keep):
    width = x.shape[-1]
    m, stride = _matrix(x, width)
    rows = m.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep else None
    param = weight if weight is not None else bias
    with _on(x) as stream:
        _check(lib().urgym_ops_layer_norm(_DTYPES[x.dtype], _DTYPES[x.dtype if param is None else param.dtype], rows, width,
                                          m.data_ptr(), stride, _ptr(weight), _ptr(bias), eps, y.data_ptr(),
                                          stats.data_ptr() if keep else None,
                                          stats.data_ptr() + 4 * rows if keep else None, stream))
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.has_bias = bias is not None
        ctx.param_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        width, L = x.shape[-1], lib()
        m, stride = _matrix(x, width)
        d, d_stride = _matrix(dy, width)
        rows = m.shape[0]
        want_w = weight is not None and ctx.needs_input_grad[1]
        want_b = ctx.has_bias and ctx.needs_input_grad[2]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(width, dtype=ctx.param_dtype, device=x.device) if want_w else None
        db = torch.empty(width, dtype=ctx.param_dtype, device=x.device) if want_b else None
        ws = None
        if want_w or want_b:
            ws = torch.empty(L.urgym_ops_layer_norm_workspace(rows, width), dtype=torch.float32, device=x.device)
        with _on(x) as stream:
            _check(L.urgym_ops_layer_norm_backward(_DTYPES[x.dtype], _DTYPES[ctx.param_dtype], rows, width, d.data_ptr(), d_stride,
                                                   m.data_ptr(), stride, _ptr(weight), stats.data_ptr(),
                                                   stats.data_ptr() + 4 * rows, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), stream))
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last axis; statistics and sums in float32.

    x: [..., width] float32, bfloat16 or float16, any strides; weight, bias: [width] of x's dtype or both float32, or None.
    Returns a contiguous tensor of x's shape and dtype.  Differentiable in x, weight and bias."""
    _need("x", x, tuple(_DTYPES))
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x of shape {tuple(x.shape)} has no last axis to normalise")
    if not eps > 0:
        raise ValueError(f"eps must be positive, not {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _need(name, p, tuple(_DTYPES), x.device)
        if p.shape != x.shape[-1:]:
            raise ValueError(f"{name} has shape {tuple(p.shape)}, x's last axis is {x.shape[-1]}")
        if p.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} is {p.dtype}: x's dtype ({x.dtype}) or float32 is needed")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype}, bias {bias.dtype}: one dtype is needed")
    _need_gpu(x)
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight is not None and weight.requires_grad
                                    or bias is not None and bias.requires_grad):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm_forward(x, weight, bias, float(eps), False)[0]


# ---- attention with a decay ----

def _need_heads(q, k, v, log_decay, dims, what):
    _need("q", q, tuple(_DTYPES))
    for name, x in (("k", k), ("v", v)):
        _need(name, x, (q.dtype,), q.device)
    if q.dim() != dims or k.shape != q.shape or v.dim() != dims or v.shape[:-1] != q.shape[:-1]:
        raise ValueError(f"q, k and v must be {what}, not {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    for name, d in (("dk", q.shape[-1]), ("dv", v.shape[-1])):
        if not 1 <= d <= MAX_HEAD_DIM:
            raise ValueError(f"{name} = {d} must be 1 .. {MAX_HEAD_DIM}")
    if q.shape[-2] < 1:
        raise ValueError("at least one head is needed")
    _need("log_decay", log_decay, (torch.float32,), q.device)
    if log_decay.shape != (q.shape[-2],):
        raise ValueError(f"log_decay has shape {tuple(log_decay.shape)}, not ({q.shape[-2]},): one value for each head")
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant of the policy: no gradient is computed for it (detach it)")


def _need_start(start, shape, device):
    if start is not None:
        _need("start", start, (torch.bool, torch.uint8), device)
        if start.shape != shape:
            raise ValueError(f"start has shape {tuple(start.shape)}, not {tuple(shape)}")


def _need_state(name, state, shape, device):
    _need(name, state, (torch.float32,), device)
    if state.shape != shape:
        raise ValueError(f"{name} has shape {tuple(state.shape)}, not {tuple(shape)}")


def _seq(q, k, v, log_decay, state, start, scale):
    steps, envs, heads, dk = q.shape
    s = _Seq(_DTYPES[q.dtype], heads, dk, v.shape[-1], steps, envs, q.data_ptr(), k.data_ptr(), v.data_ptr())
    s.q_stride[:], s.k_stride[:], s.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    s.log_decay, s.state, s.scale = log_decay.data_ptr(), _ptr(state), scale
    if start is not None:
        s.start, s.start_stride[:] = start.data_ptr(), start.stride()
    return s


def _workspace(s, backward, device):
    n = lib().urgym_ops_decay_workspace(ctypes.byref(s), backward)
    if n < 0:
        _check(-1)
    return torch.empty(n, dtype=torch.float32, device=device) if n else None


def _decay_forward(q, k, v, log_decay, state, start, scale):
    steps, envs, heads, dk = q.shape
    dv, device = v.shape[-1], q.device
    o = torch.empty((steps, envs, heads, dv), dtype=q.dtype, device=device)
    final = torch.empty((envs, heads, dk, dv), dtype=torch.float32, device=device)
    if envs:
        s = _seq(q, k, v, log_decay, state, start, scale)
        with _on(q) as stream:
            ws = _workspace(s, 0, device)
            _check(lib().urgym_ops_decay(ctypes.byref(s), o.data_ptr(), final.data_ptr(), _ptr(ws), stream))
    return o, final


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, start, scale):
        o, final = _decay_forward(q, k, v, log_decay, state, start, scale)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, log_decay, state, start)
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dfinal):
        q, k, v, log_decay, state, start = ctx.saved_tensors
        want_state = state is not None and ctx.needs_input_grad[4]
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        dstate = torch.empty_like(state) if want_state else None
        if q.shape[1]:
            do = torch.zeros((), dtype=q.dtype, device=q.device).expand(v.shape).contiguous() if do is None else _rows(do)
            dfinal = None if dfinal is None else dfinal.contiguous()
            s = _seq(q, k, v, log_decay, state, start, ctx.scale)
            with _on(q) as stream:
                ws = _workspace(s, 1, q.device)
                _check(lib().urgym_ops_decay_backward(ctypes.byref(s), do.data_ptr(), (ctypes.c_int64 * 3)(*do.stride()[:3]),
                                                      _ptr(dfinal), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dstate),
                                                      _ptr(ws), stream))
        return dq, dk, dv, None, dstate, None, None


def decay_attention(q, k, v, log_decay, state=None, start=None, scale=None):
    """Linear attention with a decay for each head, over a recorded rollout:

        S_t = exp(log_decay) S_{t-1} + k_t v_t^T   (S_{t-1} = 0 where start_t),      o_t = scale S_t^T q_t

    q, k: [steps, envs, heads, dk], v: [steps, envs, heads, dv], all float32, bfloat16 or float16, of any strides (slices of one
    projection, heads expanded from one); dk, dv up to 128.  log_decay: float32 [heads], a constant, 0 or less in use (-inf
    forgets at once).  state: float32 [envs, heads, dk, dv], what the envs remember from before (None: nothing).
    start: bool or uint8 [steps, envs], set where a new episode begins -- the step's token does not see what came before it,
    not even an infinity or NaN.  scale: 1 / sqrt(dk) if None.
    Returns (o [steps, envs, heads, dv] of q's dtype, the state after the last step).  Products are summed in float32 and
    the state stays in float32; 16-bit inputs meet scores and the carried state rounded to their own type inside the products
    for o and the gradients.  Differentiable in q, k, v and state; backward computes all three of dq, dk, dv."""
    _need_heads(q, k, v, log_decay, 4, "[steps, envs, heads, dk], the same and [steps, envs, heads, dv]")
    shape = (q.shape[1], q.shape[2], q.shape[3], v.shape[3])
    if state is not None:
        _need_state("state", state, shape, q.device)
    _need_start(start, q.shape[:2], q.device)
    _need_gpu(q)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if q.shape[0] == 0:  # no step: nothing is answered and nothing forgotten
        o = q.new_empty((0, *q.shape[1:3], v.shape[3]))
        return o, state.clone() if state is not None else torch.zeros(shape, dtype=torch.float32, device=q.device)
    q, k, v = _rows(q), _rows(k), _rows(v)
    state = None if state is None else state.contiguous()
    log_decay = log_decay.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or state is not None and state.requires_grad):
        return _DecayAttention.apply(q, k, v, log_decay, state, start, scale)
    return _decay_forward(q, k, v, log_decay, state, start, scale)


def decay_attention_step(q, k, v, log_decay, state, start=None, scale=None, state_out=None):
    """One token per env of `decay_attention`, for a rollout: q, k [envs, heads, dk], v [envs, heads, dv], state float32
    [envs, heads, dk, dv] contiguous, start bool or uint8 [envs].  The new state is written to state_out (`state` itself:
    in place; None: a new tensor).  Returns (o [envs, heads, dv], the new state).  No gradients: training runs
    `decay_attention` over the recorded steps."""
    _need_heads(q, k, v, log_decay, 3, "[envs, heads, dk], the same and [envs, heads, dv]")
    shape = (*q.shape, v.shape[2])
    _need_state("state", state, shape, q.device)
    _need_start(start, q.shape[:1], q.device)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous")
    if state_out is not None and state_out is not state:
        _need_state("state_out", state_out, shape, q.device)
        if not state_out.is_contiguous():
            raise ValueError("state_out must be contiguous")
        apart = abs(state_out.data_ptr() - state.data_ptr())
        if 0 < apart < 4 * state.numel():
            raise ValueError("state_out overlaps state without being it")
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, k, v, state)):
        raise ValueError("decay_attention_step has no gradient: call it under torch.no_grad(), or decay_attention for training")
    _need_gpu(q)
    envs, heads, dk, dv = shape
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    if state_out is None:
        state_out = torch.empty_like(state)
    o = torch.empty((envs, heads, dv), dtype=q.dtype, device=q.device)
    if envs:
        with _on(q) as stream:
            _check(lib().urgym_ops_decay_step(
                _DTYPES[q.dtype], envs, heads, dk, dv, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0),
                k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), log_decay.data_ptr(), _ptr(start),
                0 if start is None else start.stride(0), q.shape[-1] ** -0.5 if scale is None else scale, state.data_ptr(),
                state_out.data_ptr(), o.data_ptr(), stream))
    return o, state_out


__all__ = ["layer_norm", "decay_attention", "decay_attention_step", "MAX_HEAD_DIM", "SYMBOLS", "lib"]
