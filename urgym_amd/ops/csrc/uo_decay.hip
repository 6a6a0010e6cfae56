// Attention with a decay for each head: over recorded rollouts (forward, backward) and one token at a time.
//
// S_t = g keep_t S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t with g = exp(log_decay[h]), keep_t = 0 where an episode starts.
// With D_t = scale q_t do_t^T + g keep_{t+1} D_{t+1} (D_{steps} = the final state's gradient, not decayed on its way in):
//   dq_t = scale S_t do_t,   dk_t = D_t v_t,   dv_t = D_t^T k_t,   dstate = g keep_0 D_0.
// All of them are one sweep over time, o_x = sa C_x^T a_x with C_x = g C_{x-1} + sb b_x c_x^T, in other roles:
//   o : a = q,  b = k,  c = v,  forward              dq: a = do, b = v,  c = k, forward, C = S^T
//   dk: a = v,  b = do, c = q,  backward, C = D^T    dv: a = k,  b = q,  c = do, backward, C = D
// A backward sweep is a forward one with negative strides that starts at the last step.
//
// The sweep runs in chunks of up to CH = 32 tokens (16 for float32).  With C the state before the chunk, i, j inside it:
//   o_i = sa g^(i + e0) C^T a_i + sum_{j <= i} sa sb g^(i - j) (a_i . b_j) c_j
//   C  <- g^n C + sum_j sb g^(n - j - e0) b_j c_j^T         (e0 = 1 forward, 0 backward)
// which are matrix products.  A chunk ends where the next episode begins, so every chunk lies in one episode and the only mask
// is i >= j; rows past its end are zeroed by selection, so that nothing of another episode, a NaN included, is ever multiplied.
//
// One wave holds 32 columns of one (env, head)'s C in the accumulators of 16x16 matrix instructions for the whole sweep and
// needs no LDS and no barrier, because the operands' layouts meet in registers (c = lane % 16, g = lane / 16):
//   * an accumulator holds rows 4 g + r of column c; as the next product's operand its lane holds 4 elements of the contracted
//     axis at 4 g + r.  The order of a contracted axis is free as long as both sides share it, so scores (b a^T, transposed) feed
//     the product with c, and C the product with a, after a conversion only;
//   * row 4 g + r of C's tile u is dimension VA (4 g + r) + u: a lane's part of a row of a or b is then contiguous, and
//     the transposed operands (tokens contracted) are loaded as VA or VB neighbouring columns of one token per lane.
#include "uo_common.h"

typedef float f4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

struct Rows {  // one tensor [steps, envs, heads, d]
    const void* p;
    int64_t st, sn, sh;
};

struct Sweep {
    Rows a, b, c, o;  // in sweep order: a backward sweep's strides are negative, p at the last step; o is written
    int da, db;       // width of a and b, width of c and o
    const uint8_t* start;  // byte x * start_st + n * start_sn: an episode begins at token x of the sweep (NULL: none)
    int64_t start_st, start_sn;
    bool first;         // whether token 0's flag counts (a backward sweep's state enters at token 0 whatever the flags)
    const float* s_in;  // NULL: zero; element (i, j) of C at i * s_i + j * s_j, (env, head)s da * db apart
    float* s_out;       // NULL: not wanted
    const uint8_t* s_drop;  // backward: the flags [envs] (stride start_sn) that cut the state's gradient
    int s_i, s_j;
    float sa, sb, in_mul, out_mul;
    int e0;
};

struct Sweeps {
    Sweep w[3];
    unsigned count, slices, segs, heads;  // sweeps in this launch, waves for each of them and segment of the axis, segments
    unsigned items;                       // envs * heads * count * slices * segs waves
    int seg_len;                          // steps in a segment (the last may be shorter)
    int64_t steps;
    const float* log_decay;
    // segs > 1: for each wave what its segment adds to the state, or (after k_join) the state it begins with, as the wave's
    // accumulators lie in its registers; and the factor that it leaves of the state before it
    float *ws, *left;
};

template <typename T>
struct Kind;
template <>
struct Kind<float> {
    typedef f4 Frag;
    static constexpr int FE = 4;
};
template <>
struct Kind<bf16> {
    typedef bf16x8 Frag;
    static constexpr int FE = 8;
};
template <>
struct Kind<f16> {
    typedef f16x8 Frag;
    static constexpr int FE = 8;
};

// acc += a b over the fragments' contracted axis (32 deep in 16 bits, 4 x 4 in 32)
__device__ __forceinline__ f4 dot(f4 acc, bf16x8 a, bf16x8 b) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ f4 dot(f4 acc, f16x8 a, f16x8 b) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ f4 dot(f4 acc, f4 a, f4 b) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
    return acc;
}

__device__ __forceinline__ float power(float lg, int n) { return n == 0 ? 1.f : exp2f(lg * (float)n); }

// How a row's elements are fetched: EXACT: the width is the tile's and everything is 16-byte aligned; FOURS: the width and every
// offset are multiples of 4 elements; ANY: one element at a time.
enum { EXACT, FOURS, ANY };

// N elements (a power of two) at p, of which those from column col on that are below width exist
template <typename T, int N, int MODE>
__device__ __forceinline__ void fetch(T* to, const T* p, int col, int width) {
    constexpr int U = MODE == ANY ? 1 : MODE == FOURS ? (N < 4 ? N : 4) : (N * (int)sizeof(T) <= 16 ? N : 16 / (int)sizeof(T));
    typedef T V __attribute__((ext_vector_type(U)));
#pragma unroll
    for (int u = 0; u < N; u += U) {
        if constexpr (U == 1) {
            to[u] = MODE == EXACT || col + u < width ? p[u] : (T)0.f;
        } else {
            V x = (V)(T)0.f;
            if (MODE == EXACT || col + u < width) x = *(const V*)(p + u);
#pragma unroll
            for (int e = 0; e < U; e++) to[u + e] = x[e];
        }
    }
}

// N elements, or zeros where the mask is zero (a selection: nothing of what is dropped is computed with)
template <typename T, int N>
__device__ __forceinline__ void only(T* x, unsigned mask) {
    constexpr int U = 4 / sizeof(T);
    typedef T V __attribute__((ext_vector_type(U)));
#pragma unroll
    for (int i = 0; i < N; i += U) {
        if constexpr (U == 1) {
            x[i] = __uint_as_float(__float_as_uint(x[i]) & mask);
        } else {
            V v;
            v[0] = x[i], v[1] = x[i + 1];
            v = __builtin_bit_cast(V, __builtin_bit_cast(unsigned, v) & mask);
            x[i] = v[0], x[i + 1] = v[1];
        }
    }
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}

// 2^-e for a wave-wide largest magnitude in [2^e, 2^(e+1)), and 2^e; 1 for infinities and NaN.  fp16 operands are brought to about
// one by it: scores and states leave fp16's range long before the outputs do.
__device__ __forceinline__ void unit(float most, float* down, float* up) {
    unsigned e = __float_as_uint(most) & 0x7f800000u;
    if (e == 0x7f800000u || e < 0x01000000u) e = 0x3f800000u;
    *up = __uint_as_float(e);
    *down = __uint_as_float(0x7f000000u - e);
}

// element (i, j) of the state that enters the sweep
__device__ __forceinline__ float entering(const Sweep& w, unsigned nh, int i, int j) {
    return w.s_in && i < w.da && j < w.db ? w.in_mul * w.s_in[(int64_t)nh * w.da * w.db + i * w.s_i + j * w.s_j] : 0.f;
}

// element (r, u, v) of a wave's accumulators in ws: float4s, lane by lane
__device__ __forceinline__ f4* held(const Sweeps& all, unsigned item, int tiles, int tile, int lane) {
    return (f4*)all.ws + ((int64_t)item * tiles + tile) * UO_WAVE + lane;
}

// STATE: only what the segment adds to the state (no a, no o); segments after it need that before they can begin.
template <typename T, int DA, int MODE, bool STATE>
__global__ __launch_bounds__(256) void k_sweep(Sweeps all) {
    typedef typename Kind<T>::Frag Frag;
    constexpr int FE = Kind<T>::FE, NB = FE / 4, CH = 16 * NB, NF = DA / 4 / FE, VA = DA / 16, VB = 2;
    constexpr bool HALF = sizeof(T) == 2, F16 = HALF && T(1.0 / 1024 + 1) != T(1);
    unsigned item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / UO_WAVE);
    if (item >= all.items) return;
    // neighbours share their rows: the slices, then the sweeps, then the heads of one env
    unsigned slice = item % all.slices, rest = item / all.slices, role = rest % all.count, nhs = rest / all.count;
    unsigned nh = nhs / all.segs, seg = nhs % all.segs, h = nh % all.heads;
    int64_t n = nh / all.heads;
    int lane = threadIdx.x % UO_WAVE, c = lane % 16, g = lane / 16;
    const Sweep& w = all.w[role];
    int j0 = slice * 16 * VB;
    if (j0 >= w.db) return;
    const int col = j0 + VB * c, da = w.da, db = w.db;
    const int64_t x0 = (int64_t)seg * all.seg_len, left_steps = all.steps - x0;
    const int steps = left_steps < all.seg_len ? (int)left_steps : all.seg_len;
    float lg = all.log_decay[h] * 1.44269504088896340736f;

    // lane pointers: a row's part (token c), and neighbouring columns of token 4 g
    const T* pa = (const T*)w.a.p + n * w.a.sn + h * w.a.sh + (x0 + c) * w.a.st + g * (DA / 4);
    const T* pb = (const T*)w.b.p + n * w.b.sn + h * w.b.sh + (x0 + c) * w.b.st + g * (DA / 4);
    const T* pbt = (const T*)w.b.p + n * w.b.sn + h * w.b.sh + (x0 + 4 * g) * w.b.st + VA * c;
    const T* pct = (const T*)w.c.p + n * w.c.sn + h * w.c.sh + (x0 + 4 * g) * w.c.st + col;
    T* po = (T*)w.o.p + n * w.o.sn + h * w.o.sh + (x0 + 4 * g) * w.o.st + col;
    const int64_t sta = w.a.st, stb = w.b.st, stc = w.c.st, sto = w.o.st;

    f4 S[VA][VB];
#pragma unroll
    for (int u = 0; u < VA; u++)
#pragma unroll
        for (int v = 0; v < VB; v++) {
            if (STATE) {
                S[u][v] = (f4)0.f;
            } else if (all.segs > 1) {
                S[u][v] = *held(all, item, VA * VB, u * VB + v, lane);
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++) S[u][v][r] = entering(w, nh, VA * (4 * g + r) + u, col + v);
            }
        }

    // the scores' weights (i = c, j = 4 g + r; the other block of rows is 16 further), the rows' of the carried state, and the
    // tokens' on the state after a whole chunk
    float near[4], far[4], carry[NB][4], enter[FE];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        int d = c - 4 * g - r;
        near[r] = d >= 0 ? w.sa * w.sb * power(lg, d) : 0.f;
        far[r] = w.sa * w.sb * power(lg, 16 + d);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            carry[b][r] = w.sa * power(lg, 16 * b + 4 * g + r + w.e0);
            enter[4 * b + r] = w.sb * power(lg, CH - (16 * b + 4 * g + r) - w.e0);
        }
    }
    const float whole = power(lg, CH);

    // the starts of tokens [seen, seen + 128) as two words; the third window's bytes are on their way
    const uint8_t* flags = w.start ? w.start + n * w.start_sn + x0 * w.start_st : nullptr;
    const bool first = w.first || seg;
    auto flag = [&](int x) { return x < steps && (x || first) ? flags[x * w.start_st] : (uint8_t)0; };
    uint64_t m0 = 0, m1 = 0, any = 0;
    uint8_t ahead = 0;
    int seen = 0;
    if (flags) {
        uint8_t f0 = flag(lane), f1 = flag(64 + lane);
        ahead = flag(128 + lane);
        m0 = __ballot(f0 != 0), m1 = __ballot(f1 != 0);
    }

    int slow = 0;  // tokens below it are taken one at a time
    for (int x = 0; x < steps;) {
        int n_tok = steps - x < CH ? steps - x : CH;
        if (flags) {
            if (x - seen >= 64) {
                m0 = m1, m1 = __ballot(ahead != 0), seen += 64;
                ahead = flag(seen + 128 + lane);
            }
            int at = x - seen;
            uint64_t m = at ? m0 >> at | m1 << (64 - at) : m0;
            if (m & 1) {
                any = 1;
#pragma unroll
                for (int u = 0; u < VA; u++)
#pragma unroll
                    for (int v = 0; v < VB; v++) S[u][v] = (f4)0.f;
            }
            uint64_t next = m & ~1ull;
            if (next) {
                int d = __builtin_ctzll(next);
                n_tok = d < n_tok ? d : n_tok;
            }
        }
        if (x < slow) n_tok = 1;

        T ar[NB][DA / 4], br[NB][DA / 4], bt[FE][VA], ct[FE][VB];
        if (n_tok == CH) {
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (!STATE) {
                    fetch<T, DA / 4, MODE>(ar[b], pa + 16 * b * sta, g * (DA / 4), da);
                    fetch<T, DA / 4, MODE>(br[b], pb + 16 * b * stb, g * (DA / 4), da);
                }
#pragma unroll
            for (int e = 0; e < FE; e++) {
                int64_t j = e / 4 * 16 + e % 4;
                fetch<T, VA, MODE>(bt[e], pbt + j * stb, VA * c, da);
                fetch<T, VB, MODE>(ct[e], pct + j * stc, col, db);
            }
        } else {  // tokens past the chunk's end: its last one's values, replaced by zeros once all loads are on their way
            auto over = [&](int i) { return i < n_tok ? 0 : i - n_tok + 1; };
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (!STATE) {
                    int64_t at = 16 * b - over(16 * b + c);
                    fetch<T, DA / 4, MODE>(ar[b], pa + at * sta, g * (DA / 4), da);
                    fetch<T, DA / 4, MODE>(br[b], pb + at * stb, g * (DA / 4), da);
                }
#pragma unroll
            for (int e = 0; e < FE; e++) {
                int j = e / 4 * 16 + e % 4;
                int64_t at = j - over(j + 4 * g);
                fetch<T, VA, MODE>(bt[e], pbt + at * stb, VA * c, da);
                fetch<T, VB, MODE>(ct[e], pct + at * stc, col, db);
            }
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (!STATE) {
                    unsigned mask = 16 * b + c < n_tok ? ~0u : 0u;
                    only<T, DA / 4>(ar[b], mask), only<T, DA / 4>(br[b], mask);
                }
#pragma unroll
            for (int e = 0; e < FE; e++) {
                unsigned mask = e / 4 * 16 + e % 4 + 4 * g < n_tok ? ~0u : 0u;
                only<T, VA>(bt[e], mask), only<T, VB>(ct[e], mask);
            }
        }
        Frag fa[NB][NF], fb[NB][NF], fbt[VA], fct[VB];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int e = 0; e < FE; e++) fa[b][f][e] = ar[b][f * FE + e], fb[b][f][e] = br[b][f * FE + e];
#pragma unroll
        for (int e = 0; e < FE; e++) {
#pragma unroll
            for (int u = 0; u < VA; u++) fbt[u][e] = bt[e][u];
#pragma unroll
            for (int u = 0; u < VB; u++) fct[u][e] = ct[e][u];
        }

        if constexpr (!STATE) {
        // scores, transposed: row j = 4 g + r, column i = c
        float p[NB][FE];
#pragma unroll
        for (int it = 0; it < NB; it++)
#pragma unroll
            for (int jb = 0; jb < NB; jb++) {
                f4 acc = (f4)0.f;
                if (jb <= it)
#pragma unroll
                    for (int f = 0; f < NF; f++) acc = dot(acc, fb[jb][f], fa[it][f]);
#pragma unroll
                for (int r = 0; r < 4; r++) p[it][4 * jb + r] = jb < it ? acc[r] * far[r] : jb == it ? (c >= 4 * g + r ? acc[r] * near[r] : 0.f) : 0.f;
            }
        float p_down = 1.f, p_up = 1.f, s_down = 1.f, s_up = 1.f;
        if constexpr (F16) {
            float most = 0.f;
#pragma unroll
            for (int it = 0; it < NB; it++)
#pragma unroll
                for (int e = 0; e < FE; e++) most = fmaxf(most, fabsf(p[it][e]));
            unit(wave_max(most), &p_down, &p_up);
            most = 0.f;
#pragma unroll
            for (int u = 0; u < VA; u++)
#pragma unroll
                for (int v = 0; v < VB; v++)
#pragma unroll
                    for (int r = 0; r < 4; r++) most = fmaxf(most, fabsf(S[u][v][r]));
            unit(wave_max(most), &s_down, &s_up);
        }

        // o: the carried state's part, weighted by row, then the chunk's own.  Scores and state are rounded to T here: an error of
        // half a step of T in each product, as large as that of the output's own rounding.
        f4 O[NB][VB];
#pragma unroll
        for (int v = 0; v < VB; v++) {
            Frag fs[NF];
#pragma unroll
            for (int e = 0; e < DA / 4; e++) fs[e / FE][e % FE] = (T)(F16 ? S[e % VA][v][e / VA] * s_down : S[e % VA][v][e / VA]);
#pragma unroll
            for (int it = 0; it < NB; it++) {
                f4 acc = (f4)0.f;
#pragma unroll
                for (int f = 0; f < NF; f++) acc = dot(acc, fa[it][f], fs[f]);
#pragma unroll
                for (int r = 0; r < 4; r++) acc[r] *= F16 ? carry[it][r] * (s_up * p_down) : carry[it][r];
                Frag fp;
#pragma unroll
                for (int e = 0; e < FE; e++) fp[e] = (T)(F16 ? p[it][e] * p_down : p[it][e]);
                O[it][v] = dot(acc, fp, fct[v]);
            }
        }
        // A zero score times an infinity or NaN of a later token is NaN: such a chunk is done again token by token.
        if (n_tok > 1) {
            float z = 0.f;
#pragma unroll
            for (int it = 0; it < NB; it++)
#pragma unroll
                for (int v = 0; v < VB; v++)
#pragma unroll
                    for (int r = 0; r < 4; r++) z += O[it][v][r] * 0.f;
            if (__any(z != z)) {
                slow = x + n_tok;
                continue;
            }
        }
#pragma unroll
        for (int it = 0; it < NB; it++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (16 * it + 4 * g + r < n_tok) {
                    T* to = po + (int64_t)(16 * it + r) * sto;
                    if (MODE != ANY) {
                        typedef T V __attribute__((ext_vector_type(VB)));
                        V y;
#pragma unroll
                        for (int v = 0; v < VB; v++) y[v] = (T)(F16 ? O[it][v][r] * p_up : O[it][v][r]);
                        if (MODE == EXACT || col < db) *(V*)to = y;
                    } else {
#pragma unroll
                        for (int v = 0; v < VB; v++)
                            if (col + v < db) to[v] = (T)(F16 ? O[it][v][r] * p_up : O[it][v][r]);
                    }
                }

        }  // !STATE

        // the state: c weighted by its decay to the chunk's end.  In 16 bits the weighted value goes in as two parts of T, which
        // keeps the state as exact as float32 sums of this length are.  fp16 is brought to 2^14 .. 2^15 for it, where the second
        // part has its bits still, and the accumulators with it.
        float keep = whole, c_down = 1.f, c_up = 1.f;
        if (n_tok < CH) keep = power(lg, n_tok);
        if constexpr (F16) {
            float most = 0.f;
#pragma unroll
            for (int v = 0; v < VB; v++)
#pragma unroll
                for (int e = 0; e < FE; e++) most = fmaxf(most, fabsf((float)fct[v][e]));
            unit(wave_max(most), &c_down, &c_up);
            c_down *= 16384.f, c_up *= 1.f / 16384.f, keep *= c_down;
        }
#pragma unroll
        for (int v = 0; v < VB; v++) {
            Frag hi, lo;
#pragma unroll
            for (int e = 0; e < FE; e++) {
                float by = enter[e];
                if (n_tok < CH) {
                    int to = n_tok - (e / 4 * 16 + e % 4 + 4 * g) - w.e0;
                    by = w.sb * power(lg, to > 0 ? to : 0);
                }
                float y = (float)fct[v][e] * (F16 ? by * c_down : by);
                hi[e] = (T)y;
                if (HALF) lo[e] = (T)(y - (float)hi[e]);
            }
#pragma unroll
            for (int u = 0; u < VA; u++) {
                S[u][v] = dot(S[u][v] * keep, fbt[u], hi);
                if (HALF) S[u][v] = dot(S[u][v], fbt[u], lo);
                if (F16) S[u][v] *= c_up;
            }
        }
        x += n_tok;
        pa += n_tok * sta, pb += n_tok * stb, pbt += n_tok * stb, pct += n_tok * stc, po += n_tok * sto;
    }

    if (STATE) {
#pragma unroll
        for (int u = 0; u < VA; u++)
#pragma unroll
            for (int v = 0; v < VB; v++) *held(all, item, VA * VB, u * VB + v, lane) = S[u][v];
        if (lane == 0) all.left[item] = any ? 0.f : power(lg, steps);
        return;
    }
    if (!w.s_out || seg + 1 < all.segs) return;
    bool drop = w.s_drop && w.s_drop[n * w.start_sn];
#pragma unroll
    for (int u = 0; u < VA; u++)
#pragma unroll
        for (int v = 0; v < VB; v++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                int i = VA * (4 * g + r) + u;
                if (i < da && col + v < db) w.s_out[(int64_t)nh * da * db + i * w.s_i + (col + v) * w.s_j] = drop ? 0.f : w.out_mul * S[u][v][r];
            }
}

// The states that the segments begin with, from what each adds: begin_0 = what enters, begin_{s+1} = left_s begin_s + added_s
// (selected where left_s = 0, so that nothing passes a start).  A workgroup takes 32 float4s of one wave's accumulators; its 8 rows of
// threads take a run of up to 16 segments each, all of whose loads are in flight at once, then hand on through LDS.
constexpr int RUNS = 8, RUN = 16, MAX_SEGS = RUNS * RUN;

template <int DA>
__global__ __launch_bounds__(256) void k_join(Sweeps all) {
    constexpr int VA = DA / 16, VB = 2, TILES = VA * VB;
    __shared__ f4 sums[RUNS][32];
    __shared__ float lefts[RUNS];
    unsigned part = blockIdx.x % (2 * TILES), rest = blockIdx.x / (2 * TILES);
    unsigned slice = rest % all.slices, role = rest / all.slices % all.count, nh = rest / all.slices / all.count;
    const Sweep& w = all.w[role];
    if ((int)slice * 16 * VB >= w.db) return;
    int tile = part / 2, lane = part % 2 * 32 + threadIdx.x % 32, run = threadIdx.x / 32;
    unsigned per = (all.segs + RUNS - 1) / RUNS, s0 = run * per;
    auto item = [&](unsigned s) { return ((nh * all.segs + s) * all.count + role) * all.slices + slice; };
    auto step = [](f4 x, float left, f4 add) { return left == 0.f ? add : x * left + add; };
    f4 add[RUN];
    float left[RUN];
#pragma unroll
    for (unsigned i = 0; i < RUN; i++) {
        bool in = i < per && s0 + i < all.segs;
        add[i] = in ? *held(all, item(s0 + i), TILES, tile, lane) : (f4)0.f;
        left[i] = in ? all.left[item(s0 + i)] : 1.f;
    }
    f4 x = (f4)0.f;
    float l = 1.f;
#pragma unroll
    for (int i = 0; i < RUN; i++) x = step(x, left[i], add[i]), l *= left[i];
    sums[run][threadIdx.x % 32] = x;
    if (threadIdx.x % 32 == 0) lefts[run] = l;
    __syncthreads();
    int g = lane / 16, c = lane % 16, u = tile / VB, v = tile % VB;
#pragma unroll
    for (int r = 0; r < 4; r++) x[r] = entering(w, nh, VA * (4 * g + r) + u, slice * 16 * VB + VB * c + v);
    for (int i = 0; i < run; i++) x = step(x, lefts[i], sums[i][threadIdx.x % 32]);
#pragma unroll
    for (unsigned i = 0; i < RUN; i++)
        if (i < per && s0 + i < all.segs) {
            *held(all, item(s0 + i), TILES, tile, lane) = x;
            x = step(x, left[i], add[i]);
        }
}

// every access of the tensor falls on multiples of `elements` elements
static bool aligned(const Rows& r, int size, int elements) {
    return (uintptr_t)r.p % (size * elements) == 0 && r.st % elements == 0 && r.sn % elements == 0 && r.sh % elements == 0;
}

template <typename T, int DA>
static void launch(const Sweeps& s, hipStream_t st) {
    int mode = EXACT, unit = 16 / sizeof(T);
    for (int i = 0; i < s.count; i++) {
        const Sweep& w = s.w[i];
        auto all = [&](int n) { return aligned(w.a, sizeof(T), n) && aligned(w.b, sizeof(T), n) && aligned(w.c, sizeof(T), n) && aligned(w.o, sizeof(T), n); };
        if (mode == EXACT && !(w.da == DA && w.db % 32 == 0 && all(unit))) mode = FOURS;
        if (mode == FOURS && !(w.da % 4 == 0 && w.db % 4 == 0 && all(4))) mode = ANY;
    }
    unsigned grid = (s.items + 3) / 4;
    if (s.segs > 1) {
        if (mode == EXACT) k_sweep<T, DA, EXACT, true><<<grid, 256, 0, st>>>(s);
        else if (mode == FOURS) k_sweep<T, DA, FOURS, true><<<grid, 256, 0, st>>>(s);
        else k_sweep<T, DA, ANY, true><<<grid, 256, 0, st>>>(s);
        k_join<DA><<<s.items / s.segs * (DA / 16 * 2) * 2, 256, 0, st>>>(s);
    }
    if (mode == EXACT) k_sweep<T, DA, EXACT, false><<<grid, 256, 0, st>>>(s);
    else if (mode == FOURS) k_sweep<T, DA, FOURS, false><<<grid, 256, 0, st>>>(s);
    else k_sweep<T, DA, ANY, false><<<grid, 256, 0, st>>>(s);
}

template <typename T>
static void launch(const Sweeps& s, hipStream_t st) {
    if (s.w[0].da <= 32) launch<T, 32>(s, st);
    else if (s.w[0].da <= 64) launch<T, 64>(s, st);
    else launch<T, 128>(s, st);
}

static int tile(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

// The launch of `count` sweeps whose a and b fall into one tile width.  With fewer waves than fill the chip twice over (one a SIMD is
// half of that) the axis is cut into segments, at least 64 steps each: their states are computed first, then joined.
static Sweeps plan(const urgym_ops_seq* q, const Sweep* w, int count) {
    Sweeps s = {};
    s.count = count, s.heads = q->heads, s.steps = q->steps, s.log_decay = q->log_decay;
    for (int i = 0; i < count; i++) {
        s.w[i] = w[i];
        unsigned n = (w[i].db + 31) / 32;
        s.slices = n > s.slices ? n : s.slices;
    }
    s.items = (unsigned)(q->envs * q->heads) * s.count * s.slices;
    int64_t segs = s.items >= 1024 ? 1 : 2048 / s.items, most = q->steps / 64;
    segs = segs < most ? segs : most;
    segs = segs < MAX_SEGS ? segs : MAX_SEGS;
    if (segs < 2) segs = 1;
    int64_t len = (q->steps + segs - 1) / segs;
    len = (len + 31) / 32 * 32;
    s.segs = (unsigned)((q->steps + len - 1) / len), s.seg_len = (int)len;
    s.items *= s.segs;
    return s;
}

static int64_t workspace(const Sweeps& s) { return s.segs > 1 ? (int64_t)s.items * (tile(s.w[0].da) * 32 + 1) : 0; }

static void launch(const urgym_ops_seq* q, Sweeps s, float* ws, hipStream_t st) {
    s.ws = ws, s.left = ws + (int64_t)s.items * tile(s.w[0].da) * 32;
    if (q->dtype == URGYM_OPS_F32) launch<float>(s, st);
    else if (q->dtype == URGYM_OPS_BF16) launch<bf16>(s, st);
    else launch<f16>(s, st);
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

static Rows rows(const void* p, const int64_t* st) { return {p, st[0], st[1], st[2]}; }

static Rows packed(void* p, const urgym_ops_seq* s, int d) { return {p, s->envs * s->heads * d, (int64_t)s->heads * d, d}; }

static Rows reversed(Rows r, const urgym_ops_seq* s) {
    int size = s->dtype == URGYM_OPS_F32 ? 4 : 2;
    return {(const char*)r.p + (s->steps - 1) * r.st * size, -r.st, r.sn, r.sh};
}

// o (or dq with the roles changed): a, b, c in time's order from `state`
static Sweep forward(const urgym_ops_seq* s, Rows a, Rows b, Rows c, Rows o, int da, int db, bool transposed) {
    Sweep w = {};
    w.a = a, w.b = b, w.c = c, w.o = o, w.da = da, w.db = db;
    w.start = s->start, w.start_st = s->start_stride[0], w.start_sn = s->start_stride[1], w.first = true;
    w.s_in = s->state, w.s_i = transposed ? 1 : db, w.s_j = transposed ? da : 1;
    w.sa = s->scale, w.sb = 1.f, w.in_mul = 1.f, w.out_mul = 1.f, w.e0 = 1;
    return w;
}

// dk or dv: against time's order from d_state_out.  Token x of the sweep is step steps - 1 - x, which an episode border cuts from
// token x - 1 where step steps - x starts one.  A scale above 1 stays outside the state: times a c of float16 it could overflow.
static Sweep backward(const urgym_ops_seq* s, Rows a, Rows b, Rows c, Rows o, int da, int db, bool transposed, const float* d_state_out) {
    Sweep w = forward(s, reversed(a, s), reversed(b, s), reversed(c, s), reversed(o, s), da, db, transposed);
    if (s->start) w.start = s->start + s->steps * s->start_stride[0], w.start_st = -s->start_stride[0];
    w.first = false, w.e0 = 0, w.s_in = d_state_out, w.s_drop = s->start;
    if (s->scale > 1.f || s->scale < -1.f) w.sa = s->scale, w.sb = 1.f, w.in_mul = 1.f / s->scale, w.out_mul = s->scale;
    else w.sa = 1.f, w.sb = s->scale;
    return w;
}

// the launches of one direction: o's, or those of dk, dq and dv, which read the same rows and share a launch where their tiles agree
static int plans(const urgym_ops_seq* s, Rows o, Sweeps* p) {
    Sweep w = forward(s, rows(s->q, s->q_stride), rows(s->k, s->k_stride), rows(s->v, s->v_stride), o, s->dk, s->dv, false);
    p[0] = plan(s, &w, 1);
    return 1;
}

static int plans(const urgym_ops_seq* s, Rows g, const float* d_state_out, void* dq, void* dk, void* dv, float* d_state, Sweeps* p) {
    Rows q = rows(s->q, s->q_stride), k = rows(s->k, s->k_stride), v = rows(s->v, s->v_stride);
    Sweep w[3] = {backward(s, v, g, q, packed(dk, s, s->dk), s->dv, s->dk, true, d_state_out),
                  forward(s, g, v, k, packed(dq, s, s->dk), s->dv, s->dk, true),
                  backward(s, k, q, g, packed(dv, s, s->dv), s->dk, s->dv, false, d_state_out)};
    w[2].s_out = d_state;
    if (tile(s->dk) == tile(s->dv)) {
        p[0] = plan(s, w, 3);
        return 1;
    }
    p[0] = plan(s, w, 2), p[1] = plan(s, w + 2, 1);
    return 2;
}

extern "C" int64_t urgym_ops_decay_workspace(const urgym_ops_seq* s, int backward) {
    if (seq_check("urgym_ops_decay_workspace", s)) return -1;
    Sweeps p[2];
    int64_t most = 0;
    for (int i = 0, n = backward ? plans(s, Rows{}, nullptr, nullptr, nullptr, nullptr, nullptr, p) : plans(s, Rows{}, p); i < n; i++)
        most = workspace(p[i]) > most ? workspace(p[i]) : most;
    return most;
}

static int run(const char* what, const urgym_ops_seq* s, const Sweeps* p, int n, float* ws, hipStream_t st) {
    for (int i = 0; i < n; i++)
        if (workspace(p[i]) && !ws) return uo_fail("%s: a workspace is needed", what);
    for (int i = 0; i < n; i++) launch(s, p[i], ws, st);
    return uo_launched(what);
}

extern "C" int urgym_ops_decay(const urgym_ops_seq* s, void* o, float* state_out, float* ws, void* stream) {
    if (seq_check("urgym_ops_decay", s)) return -1;
    if (!o || !state_out) return uo_fail("urgym_ops_decay: o and state_out are needed");
    Sweeps p[1];
    int n = plans(s, packed(o, s, s->dv), p);
    p[0].w[0].s_out = state_out;
    return run("urgym_ops_decay", s, p, n, ws, (hipStream_t)stream);
}

extern "C" int urgym_ops_decay_backward(const urgym_ops_seq* s, const void* d_out, const int64_t d_out_stride[3],
                                        const float* d_state_out, void* dq, void* dk, void* dv, float* d_state, float* ws,
                                        void* stream) {
    if (seq_check("urgym_ops_decay_backward", s)) return -1;
    if (!d_out || !d_out_stride || !dq || !dk || !dv) return uo_fail("urgym_ops_decay_backward: d_out, dq, dk and dv are needed");
    Sweeps p[2];
    int n = plans(s, rows(d_out, d_out_stride), d_state_out, dq, dk, dv, d_state, p);
    return run("urgym_ops_decay_backward", s, p, n, ws, (hipStream_t)stream);
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
