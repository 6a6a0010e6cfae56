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

// One wave per row: the mean, then the centred second moment (no E[x^2] - mean^2, which cancels), then the output.
template <typename T, typename W>
__global__ __launch_bounds__(256) void k_norm(int64_t rows, int64_t width, const T* x, int64_t xs, const W* w, const W* b,
                                              float eps, T* y, float* mean, float* rstd) {
    int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / UO_WAVE;
    int lane = threadIdx.x % UO_WAVE;
    if (row >= rows) return;
    const T* xr = x + row * xs;
    float s = 0.f;
    for (int64_t i = lane; i < width; i += UO_WAVE) s += (float)xr[i];
    float mu = uo_wave_sum(s) / (float)width;
    float q = 0.f;
    for (int64_t i = lane; i < width; i += UO_WAVE) {
        float c = (float)xr[i] - mu;
        q += c * c;
    }
    float r = 1.0f / sqrtf(uo_wave_sum(q) / (float)width + eps);
    for (int64_t i = lane; i < width; i += UO_WAVE)
        y[row * width + i] = (T)(((float)xr[i] - mu) * r * (w ? (float)w[i] : 1.f) + (b ? (float)b[i] : 0.f));
    if (mean && lane == 0) mean[row] = mu, rstd[row] = r;
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void k_norm_dx(int64_t rows, int64_t width, const T* dy, int64_t ds, const T* x, int64_t xs,
                                                 const W* w, const float* mean, const float* rstd, T* dx) {
    int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / UO_WAVE;
    int lane = threadIdx.x % UO_WAVE;
    if (row >= rows) return;
    const T *xr = x + row * xs, *dr = dy + row * ds;
    float mu = mean[row], r = rstd[row], sg = 0.f, sh = 0.f;
    for (int64_t i = lane; i < width; i += UO_WAVE) {
        float g = (float)dr[i] * (w ? (float)w[i] : 1.f);
        sg += g;
        sh += g * (((float)xr[i] - mu) * r);
    }
    sg = uo_wave_sum(sg) / (float)width;
    sh = uo_wave_sum(sh) / (float)width;
    for (int64_t i = lane; i < width; i += UO_WAVE) {
        float g = (float)dr[i] * (w ? (float)w[i] : 1.f);
        dx[row * width + i] = (T)(r * (g - sg - ((float)xr[i] - mu) * r * sh));
    }
}

// The rows are cut into `parts` equal runs; part p's column sums go to ws[p], then k_norm_dw_sum adds the parts in order.
static int64_t norm_parts(int64_t rows) { return rows < 16 * 256 ? (rows + 15) / 16 : 256; }

template <typename T>
__global__ __launch_bounds__(64) void k_norm_dw(int64_t rows, int64_t width, const T* dy, int64_t ds, const T* x, int64_t xs,
                                                const float* mean, const float* rstd, float* ws) {
    int64_t c = (int64_t)blockIdx.y * 64 + threadIdx.x, parts = gridDim.x, p = blockIdx.x;
    if (c >= width) return;
    float dw = 0.f, db = 0.f;
    for (int64_t r = rows * p / parts; r < rows * (p + 1) / parts; r++) {
        float d = (float)dy[r * ds + c];
        dw += d * (((float)x[r * xs + c] - mean[r]) * rstd[r]);
        db += d;
    }
    ws[p * width + c] = dw;
    ws[(parts + p) * width + c] = db;
}

template <typename W>
__global__ __launch_bounds__(64) void k_norm_dw_sum(int64_t width, int64_t parts, const float* ws, W* dw, W* db) {
    int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (c >= width) return;
    float a = 0.f, b = 0.f;
    for (int64_t p = 0; p < parts; p++) a += ws[p * width + c], b += ws[(parts + p) * width + c];
    if (dw) dw[c] = (W)a;
    if (db) db[c] = (W)b;
}

static int norm_check(const char* what, int dtype, int wdtype, int64_t rows, int64_t width) {
    if (dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2) return uo_fail("%s: unknown dtype %d / %d", what, dtype, wdtype);
    if (wdtype != dtype && wdtype != URGYM_OPS_F32) return uo_fail("%s: the weight's dtype is x's or float32", what);
    if (rows < 0 || width < 1) return uo_fail("%s: rows %lld, width %lld", what, (long long)rows, (long long)width);
    if (width > (1 << 20) || rows > ((int64_t)1 << 32)) return uo_fail("%s: rows %lld x width %lld is too large", what, (long long)rows, (long long)width);
    return 0;
}

template <typename T, typename W>
static int norm_fwd(int64_t rows, int64_t width, const void* x, int64_t xs, const void* w, const void* b, float eps, void* y,
                    float* mean, float* rstd, hipStream_t st) {
    k_norm<T, W><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(rows, width, (const T*)x, xs, (const W*)w, (const W*)b, eps, (T*)y, mean, rstd);
    return uo_launched("urgym_ops_layer_norm");
}

template <typename T, typename W>
static int norm_bwd(int64_t rows, int64_t width, const void* dy, int64_t ds, const void* x, int64_t xs, const void* w,
                    const float* mean, const float* rstd, void* dx, void* dw, void* db, float* ws, hipStream_t st) {
    if (dx && rows)
        k_norm_dx<T, W><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(rows, width, (const T*)dy, ds, (const T*)x, xs, (const W*)w, mean, rstd, (T*)dx);
    if (dw || db) {
        int64_t parts = norm_parts(rows);
        unsigned cols = (unsigned)((width + 63) / 64);
        if (parts) k_norm_dw<T><<<dim3((unsigned)parts, cols), 64, 0, st>>>(rows, width, (const T*)dy, ds, (const T*)x, xs, mean, rstd, ws);
        k_norm_dw_sum<W><<<cols, 64, 0, st>>>(width, parts, ws, (W*)dw, (W*)db);
    }
    return uo_launched("urgym_ops_layer_norm_backward");
}

// calls F<T, W>(args...) for the dtype pair (wdtype is dtype or float32)
#define NORM_DISPATCH(F, ...)                                                      \
    (dtype == URGYM_OPS_F32    ? F<float, float>(__VA_ARGS__)                      \
     : dtype == URGYM_OPS_BF16 ? (wdtype ? F<bf16, bf16>(__VA_ARGS__) : F<bf16, float>(__VA_ARGS__)) \
                               : (wdtype ? F<f16, f16>(__VA_ARGS__) : F<f16, float>(__VA_ARGS__)))

extern "C" int urgym_ops_layer_norm(int dtype, int wdtype, int64_t rows, int64_t width, const void* x, int64_t x_stride,
                                    const void* weight, const void* bias, float eps, void* y, float* mean, float* rstd,
                                    void* stream) {
    if (norm_check("urgym_ops_layer_norm", dtype, wdtype, rows, width)) return -1;
    if (!rows) return 0;
    if (!x || !y || !mean != !rstd) return uo_fail("urgym_ops_layer_norm: x and y are needed, mean and rstd go together");
    return NORM_DISPATCH(norm_fwd, rows, width, x, x_stride, weight, bias, eps, y, mean, rstd, (hipStream_t)stream);
}

extern "C" int64_t urgym_ops_layer_norm_workspace(int64_t rows, int64_t width) { return rows < 0 || width < 1 ? 0 : 2 * norm_parts(rows) * width; }

extern "C" int urgym_ops_layer_norm_backward(int dtype, int wdtype, int64_t rows, int64_t width, const void* dy, int64_t dy_stride,
                                             const void* x, int64_t x_stride, const void* weight, const float* mean,
                                             const float* rstd, void* dx, void* dweight, void* dbias, float* workspace,
                                             void* stream) {
    if (norm_check("urgym_ops_layer_norm_backward", dtype, wdtype, rows, width)) return -1;
    if (rows && (!dy || !x || !mean || !rstd)) return uo_fail("urgym_ops_layer_norm_backward: dy, x, mean and rstd are needed");
    if (rows && (dweight || dbias) && !workspace) return uo_fail("urgym_ops_layer_norm_backward: a workspace is needed");
    return NORM_DISPATCH(norm_bwd, rows, width, dy, dy_stride, x, x_stride, weight, mean, rstd, dx, dweight, dbias, workspace,
                         (hipStream_t)stream);
}
