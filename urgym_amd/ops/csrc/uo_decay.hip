// Attention with a decay for each head: over recorded rollouts (forward, backward) and one token at a time.
//
// S_t = g keep_t S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t with g = exp(log_decay[h]), keep_t = 0 where an episode starts.
// With D_t = scale q_t do_t^T + g keep_{t+1} D_{t+1} (D_{steps} = the final state's gradient):
//   dq_t = scale S_t do_t,   dk_t = D_t v_t,   dv_t = D_t^T k_t,   dstate = g keep_0 D_0.
// All of them are one sweep over time, o_t = sa C_t^T a_t with C_t = g C' + sb b_t c_t^T, in other roles:
//   o : a = q,  b = k,  c = v,  forward          dq: a = do, b = v,  c = k, forward, C = S^T
//   dk: a = v,  b = do, c = q,  backward, C = D^T    dv: a = k,  b = q,  c = do, backward
#include "uo_common.h"

struct Rows {  // one tensor [steps, envs, heads, d]
    const void* p;
    int64_t st, sn, sh;
};

struct Sweep {
    Rows a, b, c, o;  // o is written
    int da, db;       // width of a and b, width of c and o
    int heads;
    int64_t steps, envs;
    const float* log_decay;
    const uint8_t* start;
    int64_t start_st, start_sn;
    const float* s_in;  // NULL: zero; element (i, j) of C at i * s_i + j * s_j, heads * envs of them, da * db apart
    float* s_out;       // NULL: not wanted
    int s_i, s_j;
    float sa, sb;
    bool reverse;
};

// One workgroup per (env, head), one thread per column of C, the column in registers; a's and b's rows pass through LDS.
template <typename T, int DA>
__global__ __launch_bounds__(128) void k_sweep(Sweep w) {
    __shared__ float rows[2][2][DA];
    int64_t n = blockIdx.x / w.heads;
    int h = blockIdx.x % w.heads, j = threadIdx.x;
    float g = expf(w.log_decay[h]), s[DA];
    const float* in = w.s_in ? w.s_in + (int64_t)blockIdx.x * w.da * w.db : nullptr;
#pragma unroll
    for (int i = 0; i < DA; i++) s[i] = in && j < w.db && i < w.da ? in[i * w.s_i + j * w.s_j] : 0.f;
    const T* a = (const T*)w.a.p + n * w.a.sn + h * w.a.sh;
    const T* b = (const T*)w.b.p + n * w.b.sn + h * w.b.sh;
    const T* c = (const T*)w.c.p + n * w.c.sn + h * w.c.sh;
    T* o = (T*)w.o.p + n * w.o.sn + h * w.o.sh;
    const uint8_t* start = w.start ? w.start + n * w.start_sn : nullptr;
    for (int64_t x = 0; x < w.steps; x++) {
        int64_t t = w.reverse ? w.steps - 1 - x : x;
        float(*row)[DA] = rows[x & 1];
        for (int i = j; i < DA; i += blockDim.x) {
            row[0][i] = i < w.da ? (float)a[t * w.a.st + i] * w.sa : 0.f;
            row[1][i] = i < w.da ? (float)b[t * w.b.st + i] * w.sb : 0.f;
        }
        __syncthreads();  // two buffers: the next step's rows are written only after every thread passed this step's barrier
        float v = j < w.db ? (float)c[t * w.c.st + j] : 0.f, acc = 0.f;
        bool fresh = w.reverse ? t + 1 < w.steps && start && start[(t + 1) * w.start_st] : start && start[t * w.start_st];
        // the gradient that enters at the last step is not decayed on its way in
        float gx = w.reverse && x == 0 ? 1.f : g;
#pragma unroll
        for (int i = 0; i < DA; i++) {
            s[i] = (fresh ? 0.f : gx * s[i]) + row[1][i] * v;
            acc += s[i] * row[0][i];
        }
        if (j < w.db) o[t * w.o.st + j] = (T)acc;
    }
    if (!w.s_out || j >= w.db) return;
    float* out = w.s_out + (int64_t)blockIdx.x * w.da * w.db;
    bool fresh = w.reverse && start && start[0];
    float gx = w.reverse ? g : 1.f;
#pragma unroll
    for (int i = 0; i < DA; i++)
        if (i < w.da) out[i * w.s_i + j * w.s_j] = fresh ? 0.f : gx * s[i];
}

template <typename T>
static void sweep(const Sweep& w, hipStream_t st) {
    unsigned grid = (unsigned)(w.envs * w.heads), block = w.db <= 64 ? 64 : 128;
    if (w.da <= 32) k_sweep<T, 32><<<grid, block, 0, st>>>(w);
    else if (w.da <= 64) k_sweep<T, 64><<<grid, block, 0, st>>>(w);
    else k_sweep<T, 128><<<grid, block, 0, st>>>(w);
}

// One wave per (env, head): lanes over the columns, the rows in turn.
template <typename T>
__global__ __launch_bounds__(64) void k_step(int heads, int dk, int dv, Rows q, Rows k, Rows v, const float* log_decay,
                                             const uint8_t* start, int64_t start_sn, float scale, const float* s_in,
                                             float* s_out, T* o) {
    int64_t n = blockIdx.x / heads;
    int h = blockIdx.x % heads;
    float g = expf(log_decay[h]);
    bool fresh = start && start[n * start_sn];
    const T *qr = (const T*)q.p + n * q.sn + h * q.sh, *kr = (const T*)k.p + n * k.sn + h * k.sh, *vr = (const T*)v.p + n * v.sn + h * v.sh;
    for (int j = threadIdx.x; j < dv; j += UO_WAVE) {
        float x = (float)vr[j], acc = 0.f;
        for (int i = 0; i < dk; i++) {
            int64_t at = ((int64_t)blockIdx.x * dk + i) * dv + j;
            float s = (fresh ? 0.f : g * s_in[at]) + (float)kr[i] * x;
            s_out[at] = s;
            acc += s * (float)qr[i];
        }
        o[(int64_t)blockIdx.x * dv + j] = (T)(scale * acc);
    }
}

static int seq_check(const char* what, int dtype, int64_t steps, int64_t envs, int heads, int dk, int dv) {
    if (dtype < 0 || dtype > 2) return uo_fail("%s: unknown dtype %d", what, dtype);
    if (dk < 1 || dk > URGYM_OPS_MAX_HEAD_DIM || dv < 1 || dv > URGYM_OPS_MAX_HEAD_DIM)
        return uo_fail("%s: dk %d and dv %d must be 1 .. %d", what, dk, dv, URGYM_OPS_MAX_HEAD_DIM);
    if (steps < 1 || envs < 1 || heads < 1) return uo_fail("%s: steps %lld, envs %lld, heads %d", what, (long long)steps, (long long)envs, heads);
    if (envs > (1 << 24) || (int64_t)heads * envs > (1 << 24) || steps > (1 << 30))
        return uo_fail("%s: steps %lld, envs %lld, heads %d is too large", what, (long long)steps, (long long)envs, heads);
    return 0;
}

static int seq_check(const char* what, const urgym_ops_seq* s) {
    if (!s) return uo_fail("%s: no sequence", what);
    if (seq_check(what, s->dtype, s->steps, s->envs, s->heads, s->dk, s->dv)) return -1;
    if (!s->q || !s->k || !s->v || !s->log_decay) return uo_fail("%s: q, k, v and log_decay are needed", what);
    return 0;
}

static Sweep base(const urgym_ops_seq* s) {
    Sweep w = {};
    w.heads = s->heads, w.steps = s->steps, w.envs = s->envs;
    w.log_decay = s->log_decay, w.start = s->start, w.start_st = s->start_stride[0], w.start_sn = s->start_stride[1];
    return w;
}

static Rows rows(const void* p, const int64_t* st) { return {p, st[0], st[1], st[2]}; }

static Rows packed(void* p, const urgym_ops_seq* s, int d) { return {p, s->envs * s->heads * d, (int64_t)s->heads * d, d}; }

static void sweep(int dtype, const Sweep& w, hipStream_t st) {
    if (dtype == URGYM_OPS_F32) sweep<float>(w, st);
    else if (dtype == URGYM_OPS_BF16) sweep<bf16>(w, st);
    else sweep<f16>(w, st);
}

extern "C" int64_t urgym_ops_decay_workspace(const urgym_ops_seq*, int) { return 0; }

extern "C" int urgym_ops_decay(const urgym_ops_seq* s, void* o, float* state_out, float*, void* stream) {
    if (seq_check("urgym_ops_decay", s)) return -1;
    if (!o || !state_out) return uo_fail("urgym_ops_decay: o and state_out are needed");
    Sweep w = base(s);
    w.a = rows(s->q, s->q_stride), w.b = rows(s->k, s->k_stride), w.c = rows(s->v, s->v_stride), w.o = packed(o, s, s->dv);
    w.da = s->dk, w.db = s->dv, w.s_in = s->state, w.s_out = state_out, w.s_i = s->dv, w.s_j = 1;
    w.sa = s->scale, w.sb = 1.f;
    sweep(s->dtype, w, (hipStream_t)stream);
    return uo_launched("urgym_ops_decay");
}

extern "C" int urgym_ops_decay_backward(const urgym_ops_seq* s, const void* d_out, const int64_t d_out_stride[3],
                                        const float* d_state_out, void* dq, void* dk, void* dv, float* d_state, float*,
                                        void* stream) {
    if (seq_check("urgym_ops_decay_backward", s)) return -1;
    if (!d_out || !d_out_stride || !dq || !dk || !dv) return uo_fail("urgym_ops_decay_backward: d_out, dq, dk and dv are needed");
    Rows q = rows(s->q, s->q_stride), k = rows(s->k, s->k_stride), v = rows(s->v, s->v_stride), g = rows(d_out, d_out_stride);
    Sweep w = base(s);
    w.a = g, w.b = v, w.c = k, w.o = packed(dq, s, s->dk);
    w.da = s->dv, w.db = s->dk, w.s_in = s->state, w.s_i = 1, w.s_j = s->dv;
    w.sa = s->scale, w.sb = 1.f;
    sweep(s->dtype, w, (hipStream_t)stream);
    w.a = v, w.b = g, w.c = q, w.o = packed(dk, s, s->dk);
    w.s_in = d_state_out, w.sa = 1.f, w.sb = s->scale, w.reverse = true;
    sweep(s->dtype, w, (hipStream_t)stream);
    w.a = k, w.b = q, w.c = g, w.o = packed(dv, s, s->dv);
    w.da = s->dk, w.db = s->dv, w.s_i = s->dv, w.s_j = 1, w.s_out = d_state;
    sweep(s->dtype, w, (hipStream_t)stream);
    return uo_launched("urgym_ops_decay_backward");
}

extern "C" int urgym_ops_decay_step(int dtype, int64_t envs, int heads, int dk, int dv, const void* q, int64_t q_sn, int64_t q_sh,
                                    const void* k, int64_t k_sn, int64_t k_sh, const void* v, int64_t v_sn, int64_t v_sh,
                                    const float* log_decay, const uint8_t* start, int64_t start_stride, float scale,
                                    const float* state, float* state_out, void* o, void* stream) {
    if (seq_check("urgym_ops_decay_step", dtype, 1, envs, heads, dk, dv)) return -1;
    if (!q || !k || !v || !log_decay || !state || !state_out || !o) return uo_fail("urgym_ops_decay_step: a pointer is missing");
    Rows rq = {q, 0, q_sn, q_sh}, rk = {k, 0, k_sn, k_sh}, rv = {v, 0, v_sn, v_sh};
    unsigned grid = (unsigned)(envs * heads);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == URGYM_OPS_F32) k_step<float><<<grid, 64, 0, st>>>(heads, dk, dv, rq, rk, rv, log_decay, start, start_stride, scale, state, state_out, (float*)o);
    else if (dtype == URGYM_OPS_BF16) k_step<bf16><<<grid, 64, 0, st>>>(heads, dk, dv, rq, rk, rv, log_decay, start, start_stride, scale, state, state_out, (bf16*)o);
    else k_step<f16><<<grid, 64, 0, st>>>(heads, dk, dv, rq, rk, rv, log_decay, start, start_stride, scale, state, state_out, (f16*)o);
    return uo_launched("urgym_ops_decay_step");
}
