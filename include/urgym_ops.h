/* urgym_ops.h -- C-ABI of the policy operators (liburgym_ops.so, gfx950).
 *
 * The operators that a policy with memory runs beside the simulator: attention with a per-head decay over recorded
 * rollouts (forward and backward, episodes packed in one time axis), its one-token form inside a rollout, and layer norm.
 *
 * Conventions (those of urgym.h): plain device pointers and sizes, no torch types.  Every call enqueues on `stream`
 * (a hipStream_t of the current device, NULL = the default stream), allocates nothing and returns immediately; it may be
 * captured into a graph.  Return 0 on success, <0 on error (message via urgym_ops_last_error, per thread); a refused call
 * has enqueued nothing.  Strides are counted in elements; the last axis of every tensor is contiguous.
 *
 * dtype codes: 0 = float32, 1 = bfloat16, 2 = float16.  States, statistics and decays are float32.
 */
#ifndef URGYM_OPS_H
#define URGYM_OPS_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define URGYM_OPS_F32 0
#define URGYM_OPS_BF16 1
#define URGYM_OPS_F16 2
#define URGYM_OPS_MAX_HEAD_DIM 128
#define URGYM_OPS_MAX_HEADS (1 << 22) /* envs * heads in one call; steps: up to 1 << 30 */

/* Message of this thread's last failed call. */
const char* urgym_ops_last_error(void);

/* y = (x - mean) * rstd * weight + bias over the last axis of x[rows, width] (row stride x_stride; y contiguous).
 * weight / bias: NULL or [width] of dtype wdtype.  mean, rstd: NULL or float32[rows], kept for the backward pass.  width up to
 * 1 << 20, rows up to 1 << 30. */
int urgym_ops_layer_norm(int dtype, int wdtype, int64_t rows, int64_t width, const void* x, int64_t x_stride,
                         const void* weight, const void* bias, float eps, void* y, float* mean, float* rstd, void* stream);

/* The float32 elements of workspace that urgym_ops_layer_norm_backward needs for the weight's and bias' gradients, whatever the types
 * and alignment. */
int64_t urgym_ops_layer_norm_workspace(int64_t rows, int64_t width);

/* dx (contiguous, NULL: not wanted), dweight, dbias (both of wdtype, NULL: not wanted) from dy[rows, width] (row stride
 * dy_stride), x, and the forward pass' mean and rstd.  The reductions run in a fixed order: repeated calls agree bit for bit. */
int urgym_ops_layer_norm_backward(int dtype, int wdtype, int64_t rows, int64_t width, const void* dy, int64_t dy_stride,
                                  const void* x, int64_t x_stride, const void* weight, const float* mean,
                                  const float* rstd, void* dx, void* dweight, void* dbias, float* workspace, void* stream);

/* A batch of `steps` x `envs` tokens with `heads` heads: q, k [steps, envs, heads, dk], v [.., dv]; element (t, n, h, d)
 * of q is at q[t * q_stride[0] + n * q_stride[1] + h * q_stride[2] + d].  start: NULL or uint8 [steps, envs], non-zero where
 * an episode begins (element strides start_stride); state: NULL (zero) or float32 [envs, heads, dk, dv], contiguous. */
typedef struct {
    int32_t dtype, heads, dk, dv;
    int64_t steps, envs;
    const void *q, *k, *v;
    int64_t q_stride[3], k_stride[3], v_stride[3];
    const float* log_decay; /* [heads] */
    const uint8_t* start;
    int64_t start_stride[2];
    const float* state;
    float scale;
} urgym_ops_seq;

/* The float32 elements of workspace (16-byte aligned) that urgym_ops_decay and urgym_ops_decay_backward need for these arguments (0:
 * none, NULL may be passed; <0: error): for copies of tensors whose rows are not whole, aligned 16-byte vectors or whose steps lie 64 MB
 * and more apart, and for the states of segments where few heads have many steps. */
int64_t urgym_ops_decay_workspace(const urgym_ops_seq* s);
int64_t urgym_ops_decay_backward_workspace(const urgym_ops_seq* s, const void* d_out, const int64_t d_out_stride[3]);

/* S_t = exp(log_decay) S_{t-1} + k_t v_t^T (S_{t-1} = 0 where start_t), o_t = scale S_t^T q_t.
 * log_decay: 0 or less.  o [steps, envs, heads, dv], state_out float32 [envs, heads, dk, dv] (S of the last step), both
 * contiguous and apart from the inputs. */
int urgym_ops_decay(const urgym_ops_seq* s, void* o, float* state_out, float* workspace, void* stream);

/* The gradients of urgym_ops_decay: from d_out (strides d_out_stride, as q's) and d_state_out (NULL: zero, contiguous) to
 * dq, dk, dv (contiguous, of dtype, all three needed) and d_state (NULL: not wanted), apart from the inputs. */
int urgym_ops_decay_backward(const urgym_ops_seq* s, const void* d_out, const int64_t d_out_stride[3],
                             const float* d_state_out, void* dq, void* dk, void* dv, float* d_state, float* workspace,
                             void* stream);

/* One token per env: q, k [envs, heads, dk], v [envs, heads, dv] (strides: env, head), start NULL or uint8 [envs] (stride
 * start_stride); state -> state_out (may be the same buffer; apart from all other inputs), o [envs, heads, dv] contiguous. */
int urgym_ops_decay_step(int dtype, int64_t envs, int heads, int dk, int dv, const void* q, int64_t q_sn, int64_t q_sh,
                         const void* k, int64_t k_sn, int64_t k_sh, const void* v, int64_t v_sn, int64_t v_sh,
                         const float* log_decay, const uint8_t* start, int64_t start_stride, float scale,
                         const float* state, float* state_out, void* o, void* stream);

#ifdef __cplusplus
}
#endif
#endif
