"""Operators of policies with memory, as HIP kernels (liburgym_ops.so, include/urgym_ops.h; for torch: urgym_ops_torch.so).

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
Drop the eager outputs first, or capture `torch.autograd.grad`.  Gradients of gradients and forward-mode gradients are not offered,
nor can a call be traced (torch.jit.trace): each is refused.
Errors: ValueError / TypeError for arguments, RuntimeError for what the library reports.  There is no CPU fallback.
"""
import importlib.util
import os

import torch  # noqa: F401

from ._native import MAX_HEAD_DIM, TORCH_PATH, missing

_ext = None


def _c():
    """the compiled operators; RuntimeError if they are not built"""
    global _ext
    if _ext is None:
        if not os.path.exists(TORCH_PATH):
            raise missing(TORCH_PATH)
        spec = importlib.util.spec_from_file_location("urgym_ops_torch", TORCH_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _ext = module
    return _ext


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last axis; statistics and sums in float32.

    x: [..., width] float32, bfloat16 or float16, any strides, width up to 1048576; weight, bias: [width] of x's dtype or both float32, or None.
    Returns a contiguous tensor of x's shape and dtype.  Differentiable in x, weight and bias."""
    return (_ext or _c()).layer_norm(x, weight, bias, eps)


def decay_attention(q, k, v, log_decay, state=None, start=None, scale=None):
    """Linear attention with a decay for each head, over a recorded rollout:

        S_t = exp(log_decay) S_{t-1} + k_t v_t^T   (S_{t-1} = 0 where start_t),      o_t = scale S_t^T q_t

    q, k: [steps, envs, heads, dk], v: [steps, envs, heads, dv], all float32, bfloat16 or float16, of any strides (slices of one
    projection, heads expanded from one); dk, dv up to 128, envs * heads up to 4194304.  log_decay: float32 [heads], a
    constant, 0 or less (-inf forgets at once; what a greater one gives is not defined).  state: float32
    [envs, heads, dk, dv], what the envs remember from before (None: nothing).  start: bool or uint8 [steps, envs], set where
    a new episode begins -- the step's token does not see what came before it, not even an infinity or NaN.  scale:
    1 / sqrt(dk) if None.
    Returns (o [steps, envs, heads, dv] of q's dtype, the state after the last step).  Products are summed in float32 and
    the state stays in float32.  Products of 16-bit inputs with scores and states take those as two bfloat16 numbers (to 2^-16,
    whatever their magnitude), three for what the state returned is a sum of; answers are rounded to their type once.
    What an infinity reaches comes out as infinity or NaN.
    Differentiable in q, k, v and state; backward computes all three of dq, dk, dv."""
    return (_ext or _c()).decay_attention(q, k, v, log_decay, state, start, scale)


def decay_attention_step(q, k, v, log_decay, state, start=None, scale=None, state_out=None):
    """One token per env of `decay_attention`, for a rollout: q, k [envs, heads, dk], v [envs, heads, dv], state float32
    [envs, heads, dk, dv] contiguous, start bool or uint8 [envs].  The new state is written to state_out (`state` itself:
    in place; None: a new tensor; another: apart from the other arguments).  Returns (o [envs, heads, dv], the new state).  No gradients: training runs
    `decay_attention` over the recorded steps."""
    return (_ext or _c()).decay_attention_step(q, k, v, log_decay, state, start, scale, state_out)


__all__ = ["layer_norm", "decay_attention", "decay_attention_step", "MAX_HEAD_DIM"]
