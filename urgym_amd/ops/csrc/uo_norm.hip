// Layer norm, forward and backward.
#include <stdarg.h>
#include <stdio.h>

#include "uo_common.h"

static thread_local char uo_message[256] = "";

int uo_fail(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(uo_message, sizeof(uo_message), fmt, ap);
    va_end(ap);
    return -1;
}

int uo_launched(const char* what) {
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : uo_fail("%s: %s", what, hipGetErrorString(e));
}

extern "C" const char* urgym_ops_last_error(void) { return uo_message; }

// A row is held by a group of G threads, K vectors of V elements each (V elements = 16 bytes, or 1 where a width, stride or
// address is odd), so x and dy are read once from memory; the statistics are the mean, then the centred second moment of the
// values in registers (E[x^2] - mean^2 would cancel).  Groups walk over the rows with the weights kept in registers and the next row
// already on its way, as it lies in memory (converted on arrival instead, its wait would come at once: 20000 x 999 in f16, 512 workgroups,
// 40 us backward, 84 so; 30 with norm_parts' workgroups).  Both directions are bound by memory: 2 (forward) and 3 (backward) row passes, 512000 x 256 in bf16 in 97 us (5.4
// TB/s) and 155 us (5.1 TB/s).
template <typename T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct Vec<T, 1> {
    typedef T type;
};

template <typename T, int V>
__device__ __forceinline__ typename Vec<T, V>::type norm_ask(const T* p) {
    return *(const typename Vec<T, V>::type*)p;
}

template <typename T, int V>
__device__ __forceinline__ void norm_take(float* to, typename Vec<T, V>::type v) {
    if constexpr (V == 1) to[0] = (float)v;
    else
#pragma unroll
        for (int e = 0; e < V; e++) to[e] = (float)v[e];
}

template <typename T, int V>
__device__ __forceinline__ void norm_load(float* to, const T* p) {
    norm_take<T, V>(to, norm_ask<T, V>(p));
}

template <typename T, int V>
__device__ __forceinline__ void norm_store(T* p, const float* from) {
    typename Vec<T, V>::type v;
    if constexpr (V == 1) v = (T)from[0];
    else
#pragma unroll
        for (int e = 0; e < V; e++) v[e] = (T)from[e];
    *(typename Vec<T, V>::type*)p = v;
}

// element i of a parameter vector of dtype wdtype, or `none` without one
__device__ __forceinline__ float norm_param(const void* w, int wdtype, int64_t i, float none) {
    return !w ? none : wdtype == URGYM_OPS_F32 ? ((const float*)w)[i] : wdtype == URGYM_OPS_BF16 ? (float)((const bf16*)w)[i] : (float)((const f16*)w)[i];
}

// elements i .. i + V - 1 of a parameter vector (16-byte aligned where V > 1)
template <typename T, int V>
__device__ __forceinline__ void norm_params(float* to, const void* w, int wdtype, int64_t i, float none) {
    if (!w) {
#pragma unroll
        for (int e = 0; e < V; e++) to[e] = none;
    } else if (wdtype == URGYM_OPS_F32) {
        constexpr int N = V < 4 ? V : 4;
#pragma unroll
        for (int e = 0; e < V; e += N) norm_load<float, N>(to + e, (const float*)w + i + e);
    } else {
        norm_load<T, V>(to, (const T*)w + i);
    }
}

// the sum over the G threads of a group, the same in all of them; G > 64: over the workgroup, through lds (two slots for each wave,
// used in turn, so one barrier a sum is enough)
template <int G>
__device__ __forceinline__ float group_sum(float x, float* lds) {
    x = uo_group_sum<G < UO_WAVE ? G : UO_WAVE>(x);
    if constexpr (G > UO_WAVE) {
        if (threadIdx.x % UO_WAVE == 0) lds[threadIdx.x / UO_WAVE] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int i = 0; i < G / UO_WAVE; i++) x += lds[i];
    }
    return x;
}

template <typename T, int G, int K, int V>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_norm(int64_t rows, int64_t width, const T* x, int64_t xs, const void* w,
                                                            const void* b, int wdtype, float eps, T* y, float* mean, float* rstd) {
    constexpr int BLOCK = G > 256 ? G : 256;
    __shared__ float lds[2][G > UO_WAVE ? G / UO_WAVE : 1];
    int t = threadIdx.x % G;
    int64_t row = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G, stride = (int64_t)gridDim.x * (BLOCK / G);
    float wv[K][V], bv[K][V];
    typename Vec<T, V>::type next[K];
    const float inv = 1.f / (float)width;
    bool have[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        int64_t i = (int64_t)(k * G + t) * V;
        have[k] = i < width, next[k] = (T)0.f;
#pragma unroll
        for (int e = 0; e < V; e++) wv[k][e] = bv[k][e] = 0.f;
        if (have[k]) {
            if (row < rows) next[k] = norm_ask<T, V>(x + row * xs + i);
            norm_params<T, V>(wv[k], w, wdtype, i, 1.f);
            norm_params<T, V>(bv[k], b, wdtype, i, 0.f);
        }
    }
    for (; row < rows; row += stride) {
        float v[K][V], s = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            norm_take<T, V>(v[k], next[k]);
#pragma unroll
            for (int e = 0; e < V; e++) s += v[k][e];
            if (have[k] && row + stride < rows) next[k] = norm_ask<T, V>(x + (row + stride) * xs + (int64_t)(k * G + t) * V);
        }
        float mu = group_sum<G>(s, lds[0]) / (float)width, q = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int e = 0; e < V; e++) {
                v[k][e] -= mu;
                if (have[k]) q += v[k][e] * v[k][e];
            }
        float r = rsqrtf(group_sum<G>(q, lds[1]) * inv + eps);
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int e = 0; e < V; e++) v[k][e] = v[k][e] * r * wv[k][e] + bv[k][e];
            if (have[k]) norm_store<T, V>(y + row * width + (int64_t)(k * G + t) * V, v[k]);
        }
        if (mean && t == 0) mean[row] = mu, rstd[row] = r;
    }
}

// dx, and in the same pass the workgroup's sums of dy xh and dy over its rows, in registers, to ws[0 / 1][workgroup][width]; the
// sums over workgroups are k_norm_dw_sum's.
template <typename T, int G, int K, int V>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_norm_back(int64_t rows, int64_t width, const T* dy, int64_t ds, const T* x,
                                                                 int64_t xs, const void* w, int wdtype, const float* mean,
                                                                 const float* rstd, T* dx, float* ws) {
    constexpr int BLOCK = G > 256 ? G : 256;
    __shared__ float lds[2][G > UO_WAVE ? G / UO_WAVE : 1];
    __shared__ float cols[G > UO_WAVE ? 1 : 2 * 4 * G * K * V];
    int t = threadIdx.x % G;
    int64_t row = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G, stride = (int64_t)gridDim.x * (BLOCK / G);
    float wv[K][V], dw[K][V], db[K][V], n_mu = 0.f, n_r = 0.f;
    typename Vec<T, V>::type nx[K], nd[K];
    const float inv = 1.f / (float)width;
    bool have[K];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            int64_t i = (int64_t)(k * G + t) * V;
            if (have[k]) nx[k] = norm_ask<T, V>(x + r * xs + i), nd[k] = norm_ask<T, V>(dy + r * ds + i);
        }
        n_mu = mean[r], n_r = rstd[r];
    };
#pragma unroll
    for (int k = 0; k < K; k++) have[k] = (int64_t)(k * G + t) * V < width, nx[k] = nd[k] = (T)0.f;
    if (row < rows) fetch(row);
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int e = 0; e < V; e++) wv[k][e] = dw[k][e] = db[k][e] = 0.f;
        if (have[k]) norm_params<T, V>(wv[k], w, wdtype, (int64_t)(k * G + t) * V, 1.f);
    }
    for (; row < rows; row += stride) {
        float h[K][V], d[K][V], mu = n_mu, r = n_r, sg = 0.f, sh = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
            norm_take<T, V>(h[k], nx[k]), norm_take<T, V>(d[k], nd[k]);
#pragma unroll
            for (int e = 0; e < V; e++) {
                h[k][e] = (h[k][e] - mu) * r;
                if (have[k]) {
                    dw[k][e] += d[k][e] * h[k][e], db[k][e] += d[k][e];
                    float gr = d[k][e] * wv[k][e];
                    sg += gr, sh += gr * h[k][e];
                }
            }
        }
        if (row + stride < rows) fetch(row + stride);
        if (!dx) continue;
        sg = group_sum<G>(sg, lds[0]) * inv;
        sh = group_sum<G>(sh, lds[1]) * inv;
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int e = 0; e < V; e++) h[k][e] = r * (d[k][e] * wv[k][e] - sg - h[k][e] * sh);
            if (have[k]) norm_store<T, V>(dx + row * width + (int64_t)(k * G + t) * V, h[k]);
        }
    }
    if (!ws) return;
    float* out = ws + (int64_t)blockIdx.x * width;
    int64_t half = (int64_t)gridDim.x * width;
    if constexpr (G > UO_WAVE) {
#pragma unroll
        for (int k = 0; k < K; k++)
            if (have[k])
#pragma unroll
                for (int e = 0; e < V; e++) {
                    int64_t i = (int64_t)(k * G + t) * V + e;
                    out[i] = dw[k][e], out[half + i] = db[k][e];
                }
    } else {  // the wave's groups first, then the four waves
        int wave = threadIdx.x / UO_WAVE;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int e = 0; e < V; e++) {
                float p = dw[k][e], q = db[k][e];
#pragma unroll
                for (int m = G; m < UO_WAVE; m *= 2) p += __shfl_xor(p, m), q += __shfl_xor(q, m);
                if (threadIdx.x % UO_WAVE < G) {
                    int i = (k * G + t) * V + e;
                    cols[wave * G * K * V + i] = p, cols[(4 + wave) * G * K * V + i] = q;
                }
            }
        __syncthreads();
        for (int i = threadIdx.x; i < width; i += BLOCK) {
            float p = 0.f, q = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) p += cols[j * G * K * V + i], q += cols[(4 + j) * G * K * V + i];
            out[i] = p, out[half + i] = q;
        }
    }
}

// Rows that no group holds (more than 4096 vectors, backward 2048 in 16 bits, or 8192 odd elements): a workgroup a row at a time, the row read again for each pass.
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_wide(int64_t rows, int64_t width, const T* x, int64_t xs, const void* w, const void* b, int wdtype,
                                                    float eps, T* y, float* mean, float* rstd) {
    __shared__ float lds[2][16];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * xs;
        float s = 0.f, q = 0.f;
        for (int64_t i = threadIdx.x; i < width; i += 1024) s += (float)xr[i];
        float mu = group_sum<1024>(s, lds[0]) / (float)width;
        for (int64_t i = threadIdx.x; i < width; i += 1024) q += ((float)xr[i] - mu) * ((float)xr[i] - mu);
        float r = 1.0f / sqrtf(group_sum<1024>(q, lds[1]) / (float)width + eps);
        for (int64_t i = threadIdx.x; i < width; i += 1024)
            y[row * width + i] = (T)(((float)xr[i] - mu) * r * norm_param(w, wdtype, i, 1.f) + norm_param(b, wdtype, i, 0.f));
        if (mean && threadIdx.x == 0) mean[row] = mu, rstd[row] = r;
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void k_norm_wide_dx(int64_t rows, int64_t width, const T* dy, int64_t ds, const T* x, int64_t xs,
                                                       const void* w, int wdtype, const float* mean, const float* rstd, T* dx) {
    __shared__ float lds[2][16];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * xs, *dr = dy + row * ds;
        float mu = mean[row], r = rstd[row], sg = 0.f, sh = 0.f;
        for (int64_t i = threadIdx.x; i < width; i += 1024) {
            float g = (float)dr[i] * norm_param(w, wdtype, i, 1.f);
            sg += g, sh += g * (((float)xr[i] - mu) * r);
        }
        sg = group_sum<1024>(sg, lds[0]) / (float)width;
        sh = group_sum<1024>(sh, lds[1]) / (float)width;
        for (int64_t i = threadIdx.x; i < width; i += 1024)
            dx[row * width + i] = (T)(r * ((float)dr[i] * norm_param(w, wdtype, i, 1.f) - sg - ((float)xr[i] - mu) * r * sh));
    }
}

template <typename T>
__global__ __launch_bounds__(64) void k_norm_wide_dw(int64_t rows, int64_t width, const T* dy, int64_t ds, const T* x, int64_t xs,
                                                     const float* mean, const float* rstd, float* ws) {
    int64_t c = (int64_t)blockIdx.y * 64 + threadIdx.x, parts = gridDim.x, p = blockIdx.x;
    if (c >= width) return;
    float dw = 0.f, db = 0.f;
    for (int64_t r = rows * p / parts; r < rows * (p + 1) / parts; r++) {
        float d = (float)dy[r * ds + c];
        dw += d * (((float)x[r * xs + c] - mean[r]) * rstd[r]), db += d;
    }
    ws[p * width + c] = dw;
    ws[(parts + p) * width + c] = db;
}

// the workgroups' sums added up in a fixed order: 32 columns by 32 runs of parts to a workgroup, the runs then through LDS (latency:
// 5 us for 256 columns of 768 parts, 4 us, 2.4 TB/s, for 5000 of 256)
__global__ __launch_bounds__(1024) void k_norm_dw_sum(int64_t width, int64_t parts, const float* ws, void* dw, void* db, int wdtype) {
    __shared__ float lds[32][33];
    void* to = blockIdx.y ? db : dw;
    if (!to) return;
    int c = threadIdx.x % 32, run = threadIdx.x / 32;
    int64_t col = (int64_t)blockIdx.x * 32 + c;
    const float* p = ws + blockIdx.y * parts * width + col;
    float s = 0.f;
    if (col < width)
#pragma unroll 8
        for (int64_t i = run; i < parts; i += 32) s += p[i * width];
    lds[run][c] = s;
    __syncthreads();
    s = uo_group_sum<32>(lds[c][run]);  // thread (run, c) sums column `run` over its 32 runs
    col = (int64_t)blockIdx.x * 32 + run;
    if (c || col >= width) return;
    if (wdtype == URGYM_OPS_F32) ((float*)to)[col] = s;
    else if (wdtype == URGYM_OPS_BF16) ((bf16*)to)[col] = (bf16)s;
    else ((f16*)to)[col] = (f16)s;
}

static int norm_check(const char* what, int dtype, int wdtype, int64_t rows, int64_t width) {
    if (dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2) return uo_fail("%s: unknown dtype %d / %d", what, dtype, wdtype);
    if (wdtype != dtype && wdtype != URGYM_OPS_F32) return uo_fail("%s: the weight's dtype is x's or float32", what);
    if (rows < 0 || width < 1) return uo_fail("%s: rows %lld, width %lld", what, (long long)rows, (long long)width);
    if (width > (1 << 20) || rows > ((int64_t)1 << 30)) return uo_fail("%s: rows %lld x width %lld is too large", what, (long long)rows, (long long)width);
    return 0;
}

// The group that holds a row of `units` vectors: one vector a thread up to a wave, then more; workgroups of 256 and 1024 threads for
// wide rows.  Single elements (odd widths) are small work a thread, so a thread takes 4 or 8 of them before the group grows.
// No group holds more than MOST.
template <bool VECTOR, int MOST, typename F>
static bool norm_group(int64_t units, F&& f) {
#define TRY(most, G, K) \
    if constexpr (most <= MOST) \
        if (units <= most) { \
            f.template operator()<G, K>(); \
            return true; \
        }
    if constexpr (VECTOR) {
        TRY(8, 8, 1) TRY(16, 16, 1) TRY(32, 32, 1) TRY(64, 64, 1) TRY(128, 64, 2) TRY(256, 256, 1) TRY(512, 256, 2) TRY(768, 256, 3)
        TRY(1024, 256, 4) TRY(2048, 1024, 2) TRY(4096, 1024, 4)
    } else {
        TRY(8, 8, 1) TRY(16, 8, 2) TRY(32, 8, 4) TRY(64, 16, 4) TRY(128, 32, 4) TRY(256, 64, 4) TRY(512, 64, 8) TRY(1024, 256, 4)
        TRY(2048, 256, 8) TRY(4096, 1024, 4) TRY(8192, 1024, 8)
    }
#undef TRY
    return false;
}

// workgroups of the forward pass (and of wide rows): enough to fill the chip, several rows each beyond that
static unsigned norm_blocks(int64_t rows, int per_block, int block) {
    int64_t n = (rows + per_block - 1) / per_block, most = 256 * 2048 / block;
    return (unsigned)(n < most ? n : most);
}

// Workgroups of the backward pass, each of which leaves a part of the column sums (two floats a column, written and read again): enough
// to have some MB of rows on the way (4 to 8 for vectors, more for the widest rows), in multiples of the 256 CUs.  `units`: a row's vectors, or 0 where it is taken by single elements.
// Backward, 48 million elements: float32, rows of 256 with 768 workgroups 115 us, 512 121, 1024 119; of 520, one to a workgroup of
// half idle threads, with 1024 129, 768 146, 512 186; of 1024 with 768 113, 512 and 1024 120; of 2048 with 512 118, 256 124; of 5000 with 256 119, 512 127;
// bf16, 1200: 1024 75, 768 82, 512 94; 2048: 768 66, 512 75; 4000: 512 73, 256 82; 8192: 256 80, 512 82.  By single elements, bf16: rows of
// 999 with 1024 83, 512 112; of 2201 with 512 98, 1024 102; of 5001 with 256 83, 512 88.
static int64_t norm_parts(int64_t rows, int64_t width, int64_t units) {
    int64_t rows_a_time = width <= 512 ? 8 : 1, n = (rows + rows_a_time - 1) / rows_a_time, most;
    if (units) most = units <= 128 ? 768 : units <= 192 ? 1024 : units <= 256 ? 768 : units <= 512 ? 512 : 256;
    else most = width <= 512 ? 768 : width <= 2048 ? 1024 : width < 4096 ? 512 : 256;
    return n < most ? n : most;
}

// the most that any type and alignment takes
static int64_t norm_most_parts(int64_t rows, int64_t width) {
    int64_t n = norm_parts(rows, width, 0);
    for (int v = 4; v <= 8; v += 4) n = norm_parts(rows, width, (width + v - 1) / v) > n ? norm_parts(rows, width, (width + v - 1) / v) : n;
    return n;
}

template <typename T, int V>
struct NormForward {
    int64_t rows, width;
    const void* x;
    int64_t xs;
    const void *w, *b;
    int wdtype;
    float eps;
    void* y;
    float *mean, *rstd;
    hipStream_t st;
    template <int G, int K>
    void operator()() {
        constexpr int block = G > 256 ? G : 256;
        k_norm<T, G, K, V><<<norm_blocks(rows, block / G, block), block, 0, st>>>(rows, width, (const T*)x, xs, w, b, wdtype, eps, (T*)y, mean, rstd);
    }
};

template <typename T, int V>
struct NormBackward {
    int64_t rows, width, parts;
    const void* dy;
    int64_t ds;
    const void* x;
    int64_t xs;
    const void* w;
    int wdtype;
    const float *mean, *rstd;
    void* dx;
    float* ws;
    hipStream_t st;
    template <int G, int K>
    void operator()() {
        constexpr int block = G > 256 ? G : 256;
        k_norm_back<T, G, K, V><<<(unsigned)parts, block, 0, st>>>(rows, width, (const T*)dy, ds, (const T*)x, xs, w, wdtype, mean, rstd, (T*)dx, ws);
    }
};

// whether rows (or, with stride 0, a parameter vector) can be read and written as 16-byte vectors of `n` elements
static bool norm_vectors(int64_t width, int64_t stride, const void* p, int n) { return width % n == 0 && stride % n == 0 && (uintptr_t)p % 16 == 0; }

template <typename T>
static int norm_fwd(int64_t rows, int64_t width, const void* x, int64_t xs, const void* w, const void* b, int wdtype, float eps, void* y,
                    float* mean, float* rstd, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool done;
    if (norm_vectors(width, xs, x, V) && norm_vectors(width, width, y, V) && norm_vectors(width, 0, w, V) && norm_vectors(width, 0, b, V))
        done = norm_group<true, 4096>(width / V, NormForward<T, V>{rows, width, x, xs, w, b, wdtype, eps, y, mean, rstd, st});
    else
        done = norm_group<false, 8192>(width, NormForward<T, 1>{rows, width, x, xs, w, b, wdtype, eps, y, mean, rstd, st});
    if (!done) k_norm_wide<T><<<norm_blocks(rows, 1, 1024), 1024, 0, st>>>(rows, width, (const T*)x, xs, w, b, wdtype, eps, (T*)y, mean, rstd);
    return uo_launched("urgym_ops_layer_norm");
}

template <typename T>
static int norm_bwd(int64_t rows, int64_t width, const void* dy, int64_t ds, const void* x, int64_t xs, const void* w, int wdtype,
                    const float* mean, const float* rstd, void* dx, void* dw, void* db, float* ws, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const bool vectors = norm_vectors(width, xs, x, V) && norm_vectors(width, ds, dy, V) && norm_vectors(width, width, dx, V) && norm_vectors(width, 0, w, V);
    const int64_t parts = norm_parts(rows, width, vectors ? width / V : 0);
    if (!dw && !db) ws = nullptr;
    if (rows && (dx || ws)) {
        // 4096 vectors of 8 elements and what the gradients need of them are more than 1024 threads' registers: 100 of each thread's
        // words lay in memory, and such rows are faster read again (bf16, 4096 x 32768: 533 us, 760 held; 4096 x 16392: 273, 536).
        // Vectors of 4 elements fit but for a few words (float32, 4096 x 16384: 228 us, 347 read again), and so do the forward pass'
        // (bf16, 4096 x 32768: 140 us, 365).
        bool done;
        if (vectors)
            done = norm_group<true, V == 8 ? 2048 : 4096>(width / V, NormBackward<T, V>{rows, width, parts, dy, ds, x, xs, w, wdtype, mean, rstd, dx, ws, st});
        else
            done = norm_group<false, 8192>(width, NormBackward<T, 1>{rows, width, parts, dy, ds, x, xs, w, wdtype, mean, rstd, dx, ws, st});
        if (!done && dx) k_norm_wide_dx<T><<<norm_blocks(rows, 1, 1024), 1024, 0, st>>>(rows, width, (const T*)dy, ds, (const T*)x, xs, w, wdtype, mean, rstd, (T*)dx);
        if (!done && ws)
            k_norm_wide_dw<T><<<dim3((unsigned)parts, (unsigned)((width + 63) / 64)), 64, 0, st>>>(rows, width, (const T*)dy, ds, (const T*)x, xs, mean, rstd, ws);
    }
    if (dw || db) k_norm_dw_sum<<<dim3((unsigned)((width + 31) / 32), 2), 1024, 0, st>>>(width, parts, ws, dw, db, wdtype);
    return uo_launched("urgym_ops_layer_norm_backward");
}

// calls F<T>(args...) for x's dtype
#define NORM_DISPATCH(F, ...) \
    (dtype == URGYM_OPS_F32 ? F<float>(__VA_ARGS__) : dtype == URGYM_OPS_BF16 ? F<bf16>(__VA_ARGS__) : F<f16>(__VA_ARGS__))

extern "C" int urgym_ops_layer_norm(int dtype, int wdtype, int64_t rows, int64_t width, const void* x, int64_t x_stride,
                                    const void* weight, const void* bias, float eps, void* y, float* mean, float* rstd,
                                    void* stream) {
    if (norm_check("urgym_ops_layer_norm", dtype, wdtype, rows, width)) return -1;
    if (!rows) return 0;
    if (!x || !y || !mean != !rstd) return uo_fail("urgym_ops_layer_norm: x and y are needed, mean and rstd go together");
    return NORM_DISPATCH(norm_fwd, rows, width, x, x_stride, weight, bias, wdtype, eps, y, mean, rstd, (hipStream_t)stream);
}

extern "C" int64_t urgym_ops_layer_norm_workspace(int64_t rows, int64_t width) { return rows < 0 || width < 1 ? 0 : 2 * norm_most_parts(rows, width) * width; }

extern "C" int urgym_ops_layer_norm_backward(int dtype, int wdtype, int64_t rows, int64_t width, const void* dy, int64_t dy_stride,
                                             const void* x, int64_t x_stride, const void* weight, const float* mean,
                                             const float* rstd, void* dx, void* dweight, void* dbias, float* workspace,
                                             void* stream) {
    if (norm_check("urgym_ops_layer_norm_backward", dtype, wdtype, rows, width)) return -1;
    if (rows && (!dy || !x || !mean || !rstd)) return uo_fail("urgym_ops_layer_norm_backward: dy, x, mean and rstd are needed");
    if (rows && (dweight || dbias) && !workspace) return uo_fail("urgym_ops_layer_norm_backward: a workspace is needed");
    return NORM_DISPATCH(norm_bwd, rows, width, dy, dy_stride, x, x_stride, weight, wdtype, mean, rstd, dx, dweight, dbias,
                         workspace, (hipStream_t)stream);
}
