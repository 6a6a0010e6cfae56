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
// which are matrix products.  Where episodes begin inside a chunk, token i sees the tokens from its own episode's first on; the
// carried state reaches the first episode's tokens and the last one's enter the new state, selected, not multiplied by zero.
// The last chunk's n tokens are the last of the CH rows, which leaves all weights but those of the carried state as they
// are; the rows before them are zeroed.  An infinity or NaN must not reach what does not see it, but times a weight of zero
// it would: a chunk with one (in c; with several episodes, in b too) is cut where the next episode begins, and if that does not
// help, into single tokens, which see nothing else.
//
// One wave (a workgroup of its own: no barrier) holds 16 VB columns of one (env, head)'s C in the accumulators of 16x16 matrix
// instructions for the whole sweep.  A chunk's operands are read out of LDS at once; while they are computed with, the next chunk's
// rows are on their way from memory into the same LDS, without passing through registers.  The operands' layouts meet
// (c = lane % 16, g = lane / 16):
//   * an accumulator holds rows 4 g + r of column c; as the next product's operand its lane holds 4 elements of the contracted
//     axis at 4 g + r.  Scores (b a^T, transposed) feed the product with c, and C the product with a, after a conversion only;
//   * o is computed transposed, so that a lane holds neighbouring columns of one token, which it stores as a vector;
//   * 16-bit operands that contract the tokens are transposed on their way out of LDS.
// LDS rows are swizzled in blocks of 16 bytes, so that both kinds of reads spread over the banks.
//
// Heads of up to 64 are bound by memory: 500 x 1024 x 4 heads of 64 in bf16 take 258 to 267 us forward (1.05 GB: 4.0 TB/s; the same loads
// and stores without the products 209 to 235) and 585 to 631 backward (dq runs against the time of dk and dv, so its inputs are read
// again: 7 reads and 3 writes, 2.62 GB, 4.2 to 4.5 TB/s; 64 columns leave 2 waves a SIMD, whose conversions of the state and the tokens to
// parts no longer hide behind them entirely: 516 to 580 with one part less for the state).  Heads of 128 are bound by the chunk's latency:
// LDS and registers leave 8 waves a CU (500 x 4096 heads, bf16: 755 us for 2.1 GB; float16, whose operands are converted too, 978).  So are
// few heads: a wave alone on its SIMD takes 4 to 5.5 us a chunk, hence the segments.
#include "uo_common.h"

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

template <int N>
struct Int {
    static constexpr int value = N;
};

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
    bool answer;  // the state is an answer, or may be: tokens enter it in three parts, whether s_out is wanted or not
    float sa, sb;
    int e0;
};

struct Sweeps {
    Sweep w[3];
    unsigned count, slices, segs, heads;  // sweeps in this launch, waves for each of them and segment of the axis, segments
    int tile, columns;                    // tile width of a and b, columns of C that a wave holds
    unsigned items;                       // envs * heads * count * slices * segs waves
    int seg_len;                          // steps in a segment (the last may be shorter)
    int64_t steps;
    const float* log_decay;
    // segs > 1: for each wave what its segment adds to the state, or (after k_join) the state it begins with, as the wave's
    // accumulators lie in its registers; and the factor that it leaves of the state before it, CUT where an episode starts in it.  Up to OWN_JOIN segments, each
    // wave joins what lies before its own.
    float *ws, *left;
};

constexpr unsigned OWN_JOIN = 8;
constexpr float CUT = -1.f;  // (not zero: a decay may underflow to that, and then still hands on an infinity or NaN)

template <typename T>
struct Kind {
    static constexpr bool HALF = sizeof(T) == 2, F16 = __is_same(T, f16);
};
// the numbers of bfloat16 (float32's range) that hold an element of T exactly: its operands' parts in products with what is computed
template <typename T>
constexpr int PARTS = Kind<T>::F16 ? 2 : 1;
template <typename T>
struct FragOf {
    typedef f4 type;
};
template <>
struct FragOf<bf16> {
    typedef bf16x8 type;
};
template <>
struct FragOf<f16> {
    typedef f16x8 type;
};
// operands of products with what is computed
template <typename T>
struct PartOf {
    typedef bf16x8 type;
};
template <>
struct PartOf<float> {
    typedef f4 type;
};

// A wave's tiles in LDS: CH tokens of a and b (DA wide) and of 16 VB columns of c
template <typename T, int DA_, int VB_>
struct Tile {
    static constexpr int DA = DA_, VB = VB_, ES = sizeof(T), FE = 16 / ES, NB = FE / 4, CH = 16 * NB, NF = DA / 4 / FE, VA = DA / 16;
    static constexpr int RA = DA * ES, RC = 16 * VB * ES;  // bytes of a row
    static constexpr int A0 = 0, B0 = CH * RA, C0 = 2 * CH * RA, BUF = 2 * CH * RA + CH * RC;
    // the dimension of row m of C's tile u, and the column (of the wave's) of its column m of tile v: in 16 bits 4 + 4 elements of
    // two tiles are 16 neighbouring bytes, in 32 the tiles' elements alternate
    static __device__ __forceinline__ int dim(int u, int m) { return ES == 2 ? 32 * (u / 2) + 8 * (m / 4) + 4 * (u % 2) + m % 4 : VA * m + u; }
    static __device__ __forceinline__ int col(int v, int m) { return ES == 2 ? 32 * (v / 2) + 8 * (m / 4) + 4 * (v % 2) + m % 4 : VB * m + v; }
};

// where byte `byte` of row t lies in a tile of RB bytes a row: blocks of 16 bytes are exchanged so that 8 rows' blocks of one column
// of blocks fall on 8 different places of 128 bytes (reads of rows), and 4 rows' four blocks on two of each (transposed reads)
template <int RB>
__device__ __forceinline__ int place(int t, int byte) {
    constexpr int N = RB / 16;
    int s = N >= 8 ? (t & 1) << 2 | (t >> 1 & 3) : t / 2 % 4;
    return t * RB + ((byte / 16 ^ s) * 16) + byte % 16;
}

// acc += a b over the fragments' contracted axis (32 deep in 16 bits, 4 x 4 in 32)
__device__ __forceinline__ f4 dot(f4 acc, bf16x8 a, bf16x8 b) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ f4 dot(f4 acc, f16x8 a, f16x8 b) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ f4 dot(f4 acc, f4 a, f4 b) {
#pragma unroll
    for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
    return acc;
}

// acc += x y for factors in parts, the largest first, but for products of two parts below what the sums of parts leave out
template <class P, int X, int Y>
__device__ __forceinline__ f4 dots(f4 acc, const P (&x)[X], const P (&y)[Y]) {
    constexpr int MOST = X > Y ? X : Y;
#pragma unroll
    for (int i = 0; i < X; i++)
#pragma unroll
        for (int j = 0; j < Y && i + j < MOST; j++) acc = dot(acc, x[i], y[j]);
    return acc;
}

// 2^(lg n); 1 for n = 0, whatever lg
__device__ __forceinline__ float power(float lg, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(lg * (float)n); }

// N elements at an address that need not be a vector's
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Piece {
    T __attribute__((ext_vector_type(N))) v;
};

// Columns col .. of the row of `width` elements at p as 16 bytes, zeros where they do not exist.  A piece that leaves the row is the
// row's last 16 bytes, moved to their places; in rows of less than that each element is clamped.
template <typename T>
__device__ __forceinline__ u4 padded(const T* p, int col, int width) {
    constexpr int N = 16 / sizeof(T);
    u4 x;
    if (width >= N) {
        x = __builtin_bit_cast(u4, ((const Piece<T, N>*)(p + (col < width - N ? col : width - N)))->v);
        int over = col - (width - N);  // elements to move down by
        if (over >= N) return (u4)0u;
        over = over < 0 ? 0 : over;
        if (over & (N / 2)) x = u4{x[2], x[3], 0u, 0u};
        if (over & (N / 4)) x = u4{x[1], x[2], x[3], 0u};
        if (N == 8 && (over & 1)) x = u4{x[0] >> 16 | x[1] << 16, x[1] >> 16 | x[2] << 16, x[2] >> 16 | x[3] << 16, x[3] >> 16};
        return x;
    }
    T y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = p[col + i < width ? col + i : width - 1];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) x[i] = col + i < width ? __builtin_bit_cast(unsigned, y[i]) : 0u;
        else x[i] = (col + 2 * i < width ? __builtin_bit_cast(uint16_t, y[2 * i]) : 0u) | (col + 2 * i + 1 < width ? (unsigned)__builtin_bit_cast(uint16_t, y[2 * i + 1]) << 16 : 0u);
    }
    return x;
}

// Tensors whose rows the sweeps cannot load as aligned vectors (odd widths, odd addresses, a chunk over more than 2 GiB) are first
// copied, rows padded to whole vectors: it costs their bytes three times, but the sweep then runs at its full rate (65 wide heads,
// bf16, 103 x 1151 x 8: forward 3.2 ms with rows fetched through registers in the sweep).  A copy in time's order whose chunks lay as
// far apart has each head's steps together instead.
struct Packs {
    struct {
        Rows from, to;
        int width;
    } t[4];
    int count;
    unsigned heads, envs;
    int64_t steps;
};

template <typename T>
__global__ __launch_bounds__(256) void k_pack(Packs p) {
    constexpr int N = 16 / sizeof(T);
    const auto& w = p.t[blockIdx.z];
    const unsigned pieces = (w.width + N - 1) / N, i = blockIdx.x * 256 + threadIdx.x, row = i / pieces, n = row / p.heads, h = row % p.heads;
    if (n >= p.envs) return;
    const int col = i % pieces * N;
    const T* from = (const T*)w.from.p + n * w.from.sn + h * w.from.sh;
    T* to = (T*)w.to.p + n * w.to.sn + h * w.to.sh + col;
    for (int64_t t = blockIdx.y; t < p.steps; t += gridDim.y) *(u4*)(to + t * w.to.st) = padded(from + t * w.from.st, col, w.width);
}

// 16 bytes at base + each lane's offset to LDS bytes to .. to + 1023, lane by lane.  Written as assembly because the compiler would
// wait for it before the next read of LDS; the waits are `landed`.  m0 is the address in LDS, and its old value is lost.  (The compiler
// warns of m0 among the clobbers, that it may not be preserved: that is what is said.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(unsigned to, const void* base, unsigned offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Fragments from LDS, as words.  `row`: row t of a tile, the f-th part of it (operand with the dimensions contracted);
// `columns`: N tiles of its columns with the tokens contracted.
template <class L, int RB>
__device__ __forceinline__ u4 row(const char* tile, int t, int f, int g) {
    return *(const u4*)(tile + place<RB>(t, L::ES == 2 ? 64 * f + 16 * g : g * (RB / 4) + 16 * f));
}

template <class L, int RB, int N>
__device__ __forceinline__ void columns(u4* to, const char* tile, int c, int g) {
    if constexpr (L::ES == 2) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4* P;
#pragma unroll
        for (int u = 0; u < N; u++) {
            const char* at = tile + place<RB>(4 * g + c / 4, 64 * (u / 2) + 16 * (c % 4) + 8 * (u % 2));
            u2 lo = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at)));
            u2 hi = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(at + 16 * RB)));
            to[u] = u4{lo[0], lo[1], hi[0], hi[1]};
        }
    } else {
        constexpr int W = N < 4 ? N : 4;
        typedef unsigned V __attribute__((ext_vector_type(W)));
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int u = 0; u < N; u += W) {
                V x = *(const V*)(tile + place<RB>(4 * g + r, (N * c + u) * 4));
#pragma unroll
                for (int e = 0; e < W; e++) to[u + e][r] = x[e];
            }
    }
}

// N parts of a fragment of float32 numbers, each the rest after those before it, rounded; y becomes what is left.  (The pair is
// opaque to the compiler, which would convert each of the two by itself as well.)
template <int N>
__device__ __forceinline__ void split(f4 (&to)[N], float (&y)[4]) {
    static_assert(N == 1);
    to[0] = f4{y[0], y[1], y[2], y[3]};
}
template <int N>
__device__ __forceinline__ void split(bf16x8 (&to)[N], float (&y)[8]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        u4 pairs;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
            unsigned w = __builtin_bit_cast(unsigned, bf16x2{(bf16)y[e], (bf16)y[e + 1]});
            asm("" : "+v"(w));
            y[e] -= __uint_as_float(w << 16), y[e + 1] -= __uint_as_float(w & 0xffff0000u);
            pairs[e / 2] = w;
        }
        to[i] = __builtin_bit_cast(bf16x8, pairs);
    }
}

// y, rounded here: a product fused into a subtraction of split() would give that another y
__device__ __forceinline__ float rounded(float y) {
    asm("" : "+v"(y));
    return y;
}

// The operand x of a product with what is computed, as numbers of bfloat16 whose sum it is: float16 takes two (8 bits and the 3 that
// are left).  What is computed is rounded to bfloat16's parts, whose range is float32's, never to float16: scores and states leave that
// range, and no one scale brings columns, tokens and dimensions of very different magnitudes into it.
__device__ __forceinline__ void parts_of(bf16x8 (&to)[1], bf16x8 x) { to[0] = x; }
__device__ __forceinline__ void parts_of(f4 (&to)[1], f4 x) { to[0] = x; }
__device__ __forceinline__ void parts_of(bf16x8 (&to)[2], f16x8 x) {
    u4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float y[2], l[2];
#pragma unroll
        for (int e = 0; e < 2; e++) y[e] = (float)x[2 * i + e], l[e] = y[e] - __uint_as_float(__float_as_uint(y[e]) & 0xffff0000u);
        hi[i] = __builtin_amdgcn_perm(__float_as_uint(y[1]), __float_as_uint(y[0]), 0x07060302u);  // both upper halves
        lo[i] = __builtin_amdgcn_perm(__float_as_uint(l[1]), __float_as_uint(l[0]), 0x07060302u);
    }
    to[0] = __builtin_bit_cast(bf16x8, hi), to[1] = __builtin_bit_cast(bf16x8, lo);
}

// element (i, j) of the state that enters the sweep
__device__ __forceinline__ float entering(const Sweep& w, unsigned nh, int i, int j) {
    return w.s_in && i < w.da && j < w.db ? w.s_in[(int64_t)nh * w.da * w.db + i * w.s_i + j * w.s_j] : 0.f;
}

// All of a lane's elements of the state at p, unscaled, or to p: as vectors where its elements are neighbours, the tiles are full and p
// is 16-byte aligned.  p: the state of this (env, head).
template <class L>
__device__ __forceinline__ bool vectors(const Sweep& w, const float* p) {
    return w.da == L::DA && w.db % (16 * L::VB) == 0 && (uintptr_t)p % 16 == 0;
}

template <class L>
__device__ __forceinline__ void state_load(f4 (&S)[L::VA][L::VB], const Sweep& w, const float* p, int j0, int c, int g) {
    constexpr int VA = L::VA, VB = L::VB;
    const bool full = vectors<L>(w, p);
    if (full && w.s_i == 1) {  // columns lie in a row: 4 neighbouring dimensions (16 bits), or all 4 VA of them
#pragma unroll
        for (int v = 0; v < VB; v++) {
            const float* q = p + (int64_t)(j0 + L::col(v, c)) * w.s_j;
#pragma unroll
            for (int i = 0; i < VA; i++) {
                f4 x = *(const f4*)(q + (L::ES == 2 ? L::dim(i, 4 * g) : 4 * VA * g + 4 * i));
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (L::ES == 2) S[i][v][e] = x[e];
                    else S[(4 * i + e) % VA][v][(4 * i + e) / VA] = x[e];
                }
            }
        }
    } else if (full && L::ES == 4) {  // rows, of which a lane has VB neighbours
        typedef float V __attribute__((ext_vector_type(VB)));
#pragma unroll
        for (int u = 0; u < VA; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                V x = *(const V*)(p + (int64_t)L::dim(u, 4 * g + r) * w.s_i + j0 + VB * c);
#pragma unroll
                for (int v = 0; v < VB; v++) S[u][v][r] = x[v];
            }
    } else {
#pragma unroll
        for (int u = 0; u < VA; u++)
#pragma unroll
            for (int v = 0; v < VB; v++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    int i = L::dim(u, 4 * g + r), j = j0 + L::col(v, c);
                    S[u][v][r] = i < w.da && j < w.db ? p[(int64_t)i * w.s_i + (int64_t)j * w.s_j] : 0.f;
                }
    }
}

template <class L>
__device__ __forceinline__ void state_store(const f4 (&S)[L::VA][L::VB], float by, bool drop, const Sweep& w, float* p, int j0, int c, int g) {
    constexpr int VA = L::VA, VB = L::VB;
    const bool full = L::ES == 4 && w.s_j == 1 && vectors<L>(w, p);
#pragma unroll
    for (int u = 0; u < VA; u++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            int i = L::dim(u, 4 * g + r);
            if (full) {
                typedef float V __attribute__((ext_vector_type(VB)));
                V x;
#pragma unroll
                for (int v = 0; v < VB; v++) x[v] = drop ? 0.f : by * S[u][v][r];
                *(V*)(p + (int64_t)i * w.s_i + j0 + VB * c) = x;
            } else {
#pragma unroll
                for (int v = 0; v < VB; v++) {
                    int j = j0 + L::col(v, c);
                    if (i < w.da && j < w.db) p[(int64_t)i * w.s_i + (int64_t)j * w.s_j] = drop ? 0.f : by * S[u][v][r];
                }
            }
        }
}

// element (r, u, v) of a wave's accumulators in ws: float4s, lane by lane
__device__ __forceinline__ f4* held(const Sweeps& all, unsigned item, int tiles, int tile, int lane) {
    return (f4*)all.ws + ((int64_t)item * tiles + tile) * UO_WAVE + lane;
}

// the state after a segment that leaves `left` of x and adds `add` (selected: nothing passes a start)
__device__ __forceinline__ f4 joined(f4 x, float left, f4 add) { return left == CUT ? add : x * left + add; }

// STATE: only what the segment adds to the state (no a, no o); segments after it need that before they can begin.
// Two waves a SIMD at least, that is 256 registers at most: then matrix instructions accumulate in ordinary registers, where C is
// scaled and converted between any two of them.
template <typename T, class L, bool STATE>
__global__ __launch_bounds__(64, 2) void k_sweep(Sweeps all) {
    typedef typename FragOf<T>::type Frag;
    typedef typename PartOf<T>::type Part;
    constexpr int FE = L::FE, NB = L::NB, CH = L::CH, NF = L::NF, VA = L::VA, VB = L::VB, RA = L::RA, RC = L::RC;
    constexpr bool HALF = Kind<T>::HALF;
    constexpr int P = PARTS<T>, TWO = HALF ? 2 : 1;
    __shared__ __attribute__((aligned(256))) char lds[L::BUF];
    // workgroups go to the 8 XCDs in turn: each takes a run of items, for neighbours share rows -- the slices, then the sweeps,
    // then the heads of one env -- and their L2
    unsigned item = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
    if (item >= all.items) return;
    unsigned slice = item % all.slices, rest = item / all.slices, role = rest % all.count, nhs = rest / all.count;
    unsigned nh = nhs / all.segs, seg = nhs % all.segs, h = nh % all.heads;
    int64_t n = nh / all.heads;
    const int lane = threadIdx.x, c = lane % 16, g = lane / 16;
    const Sweep& w = all.w[role];
    const int j0 = slice * 16 * VB, da = w.da, db = w.db;
    if (j0 >= db) return;
    const int64_t x0 = (int64_t)seg * all.seg_len, left_steps = all.steps - x0;
    const int steps = left_steps < all.seg_len ? (int)left_steps : all.seg_len;
    const float lg = all.log_decay[h] * 1.44269504088896340736f;
    const T* const pa = (const T*)w.a.p + n * w.a.sn + h * w.a.sh + x0 * w.a.st;
    const T* const pb = (const T*)w.b.p + n * w.b.sn + h * w.b.sh + x0 * w.b.st;
    const T* const pc = (const T*)w.c.p + n * w.c.sn + h * w.c.sh + x0 * w.c.st + j0;
    const int64_t sta = w.a.st, stb = w.b.st, stc = w.c.st, sto = w.o.st;
    // o: token c, the lane's run of 4 VB columns (float32) or its runs of 8 (16 bits: one in every 32)
    T* const po = (T*)w.o.p + n * w.o.sn + h * w.o.sh + (x0 + c) * sto + j0 + (HALF ? 8 : 4 * VB) * g;

    // (Everything that has to come from memory is asked for first: the starts, the state, the first chunk.)
    // the starts of tokens [seen, seen + 128) as two words; the third window's bytes are on their way
    const uint8_t* flags = w.start ? w.start + n * w.start_sn + x0 * w.start_st : nullptr;
    const bool first = w.first || seg;
    auto flag = [&](int x) { return x < steps && (x || first) ? flags[x * w.start_st] : (uint8_t)0; };
    uint64_t m0 = 0, m1 = 0, any = 0;
    uint8_t f0 = 0, f1 = 0, ahead = 0;
    int seen = 0;
    if (flags) f0 = flag(lane), f1 = flag(64 + lane), ahead = flag(128 + lane);

    // C = unit * S: a chunk's decay goes into the unit, and into the tokens that enter, instead of into all of S
    f4 S[VA][VB];
    float s_unit = 1.f;
#pragma unroll
    for (int u = 0; u < VA; u++)
#pragma unroll
        for (int v = 0; v < VB; v++) S[u][v] = !STATE && all.segs > OWN_JOIN ? *held(all, item, VA * VB, u * VB + v, lane) : (f4)0.f;
    if (!STATE && all.segs <= OWN_JOIN && w.s_in) state_load<L>(S, w, w.s_in + (int64_t)nh * da * db, j0, c, g);
    if (!STATE && all.segs <= OWN_JOIN) {
        for (unsigned before = seg; before; before--) {
            unsigned other = item - before * all.count * all.slices;
            float left = all.left[other];
#pragma unroll
            for (int u = 0; u < VA; u++)
#pragma unroll
                for (int v = 0; v < VB; v++) S[u][v] = joined(S[u][v], left, *held(all, other, VA * VB, u * VB + v, lane));
        }
    }

    if (flags) m0 = __ballot(f0 != 0), m1 = __ballot(f1 != 0);

    // the scores' weights (i = c, j = 4 g + r; the other block of rows is 16 further), the rows' of the carried state, and the
    // tokens' on the state after a whole chunk
    float near[4], far[4], carry[NB], enter[FE], whole;
    int slow = 0, cut = 0;  // tokens below `slow` are taken one at a time, chunks below `cut` end with their episode
    // the chunk that begins at token x: its length, whether an episode begins with it, and the tokens inside it that begin one
    auto chunk = [&](int x, bool* fresh, unsigned* inside) {
        int n_tok = x < slow ? 1 : steps - x < CH ? steps - x : CH;
        *fresh = false, *inside = 0;
        if (flags) {
            int at = x - seen;
            uint64_t m = at == 0 ? m0 : at < 64 ? m0 >> at | m1 << (64 - at) : m1 >> (at - 64);
            *fresh = m & 1;
            unsigned next = (unsigned)m & (unsigned)((1ull << n_tok) - 2);
            if (next && x < cut) n_tok = __builtin_ctz(next);
            else *inside = next;
        }
        return n_tok;
    };

    // A chunk's rows into LDS, lane by lane 16 bytes; the rows before a short chunk's are its first one's, zeroed before they are used.
    // What lies beyond a row's last vector is not loaded and stays zero.  Offsets are unsigned: from a load's lowest row, which in
    // a backward sweep is the last.
    const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    auto load_rows = [&](auto size, auto whole, const T* base, int64_t st, int tile0, int width, int x, int n_tok) {
        constexpr int RB = decltype(size)::value, K = CH * RB / 1024, ROWS = 1024 / RB;  // rows of one load
        const int l = lane / (RB / 16);
        const unsigned stride = (unsigned)(st < 0 ? -st : st) * sizeof(T);
#pragma unroll
        for (int k = 0; k < K; k++) {
            int t = k * ROWS + l, ts = ROWS % 8 ? t : l;
            int byte = place<RB>(ts, lane * 16 % RB) - ts * RB;  // exchanging blocks twice is nothing: what belongs at this place
            int tt = n_tok == CH ? t : t < CH - n_tok ? 0 : t - (CH - n_tok);
            int low = n_tok == CH ? k * ROWS : 0, row = n_tok == CH ? l : tt, last = n_tok == CH ? ROWS - 1 : n_tok - 1;
            const T* from = base + (int64_t)(x + low + (st < 0 ? last : 0)) * st;
            if (decltype(whole)::value || byte < width * (int)sizeof(T)) load_to_lds(at + tile0 + k * 1024, from, (unsigned)(st < 0 ? last - row : row) * stride + byte);
        }
    };
    auto rows_of = [&](auto size, const T* base, int64_t st, int tile0, int width, int x, int n_tok) {
        if (width * (int)sizeof(T) >= decltype(size)::value) load_rows(size, Int<1>(), base, st, tile0, width, x, n_tok);
        else load_rows(size, Int<0>(), base, st, tile0, width, x, n_tok);
    };
    auto issue = [&](int x, int n_tok) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every read has been answered
        if (!STATE) rows_of(Int<RA>(), pa, sta, L::A0, da, x, n_tok);
        rows_of(Int<RA>(), pb, stb, L::B0, da, x, n_tok);
        rows_of(Int<RC>(), pc, stc, L::C0, db - j0, x, n_tok);
    };

    // One chunk: the operands from LDS, then (`next`: the next chunk's loads begin) o and the state, then (`done`: they have landed)
    // the stores.  False, and nothing done, where the chunk has to be taken in parts.
    auto compute = [&](int x, int n_tok, bool fresh, unsigned inside, auto next, auto done) {
        char* buf = lds;
        if (n_tok < CH) {
            auto zero = [&](auto size, int tile0) {
                constexpr int RB = decltype(size)::value;
#pragma unroll
                for (int k = 0; k < CH * RB / 1024; k++)
                    if (k * (1024 / RB) + lane / (RB / 16) < CH - n_tok) *(u4*)(buf + tile0 + k * 1024 + lane * 16) = (u4)0u;
            };
            if (!STATE) zero(Int<RA>(), L::A0);
            zero(Int<RA>(), L::B0), zero(Int<RC>(), L::C0);
        }
        u4 wct[VB];
        columns<L, RC, VB>(wct, buf + L::C0, c, g);
        Frag fct[VB];
#pragma unroll
        for (int v = 0; v < VB; v++) fct[v] = __builtin_bit_cast(Frag, wct[v]);
        // (whether there is an infinity or NaN, the product with a matrix of zeros tells)
        if (n_tok > 1 && (!STATE || inside)) {
            float z = 0.f;
#pragma unroll
            for (int v = 0; v < VB; v++) z += dot((f4)0.f, (Frag)(T)0.f, fct[v])[0];
            if (__any(z != z)) return false;
        }
        Frag fa[STATE ? 1 : NB][NF], fb[STATE ? 1 : NB][NF], fbt[VA];
        if constexpr (!STATE)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int f = 0; f < NF; f++) {
                    fa[b][f] = __builtin_bit_cast(Frag, row<L, RA>(buf + L::A0, 16 * b + c, f, g));
                    fb[b][f] = __builtin_bit_cast(Frag, row<L, RA>(buf + L::B0, 16 * b + c, f, g));
                }
        u4 wbt[VA];
        columns<L, RA, VA>(wbt, buf + L::B0, c, g);
#pragma unroll
        for (int u = 0; u < VA; u++) fbt[u] = __builtin_bit_cast(Frag, wbt[u]);
        // the row from which on row i's episode lies in the chunk (0: from before it), and the last row's
        int from[NB], last = 0;
#pragma unroll
        for (int b = 0; b < NB; b++) from[b] = 0;
        if (inside) {
            float z = 0.f;
#pragma unroll
            for (int u = 0; u < VA; u++) z += dot((f4)0.f, (Frag)(T)0.f, fbt[u])[0];
            if (__any(z != z)) return false;
            unsigned begins = inside << (CH - n_tok);
            last = 31 - __builtin_clz(begins);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                unsigned before = begins & (2u << (16 * b + c)) - 1;
                from[b] = before ? 31 - __builtin_clz(before) : 0;
            }
        }
        next();
        if (fresh) {
            any = 1, s_unit = 1.f;
#pragma unroll
            for (int u = 0; u < VA; u++)
#pragma unroll
                for (int v = 0; v < VB; v++) S[u][v] = (f4)0.f;
        }

        f4 O[NB][VB];
        if constexpr (!STATE) {
            // scores, transposed: row j = 4 g + r, column i = c
            f4 sc[NB][NB];
#pragma unroll
            for (int jb = 0; jb < NB; jb++)
#pragma unroll
                for (int f = 0; f < NF; f++)
#pragma unroll
                    for (int it = jb; it < NB; it++) sc[it][jb] = dot(f ? sc[it][jb] : (f4)0.f, fb[jb][f], fa[it][f]);
            float p[NB][FE];
#pragma unroll
            for (int it = 0; it < NB; it++)
#pragma unroll
                for (int jb = 0; jb < NB; jb++)
#pragma unroll
                    for (int r = 0; r < 4; r++) p[it][4 * jb + r] = jb < it ? sc[it][jb][r] * far[r] : jb == it && c >= 4 * g + r ? sc[it][jb][r] * near[r] : 0.f;
            if (inside)
#pragma unroll
                for (int it = 0; it < NB; it++)
#pragma unroll
                    for (int e = 0; e < FE; e++) p[it][e] = e / 4 * 16 + e % 4 + 4 * g >= from[it] ? p[it][e] : 0.f;

            // o, transposed: the carried state's part, weighted by token, then the chunk's own.  16-bit operands meet scores and states
            // as two numbers of bfloat16 (2^-16), so that the output's own rounding is what is left.  (500 x 1024 x 4 heads of 64, bf16: 276 us
            // forward and 620 backward with one number for the state, 277 and 650 so.)
            Part fp[NB][TWO];
#pragma unroll
            for (int it = 0; it < NB; it++)
#pragma unroll
                for (int e = 0; e < FE; e++) p[it][e] = rounded(p[it][e]);
#pragma unroll
            for (int it = 0; it < NB; it++) split(fp[it], p[it]);
            float by_token[NB];
#pragma unroll
            for (int it = 0; it < NB; it++) by_token[it] = carry[it] * s_unit;
            if (n_tok < CH)
#pragma unroll
                for (int it = 0; it < NB; it++) {
                    int i = 16 * it + c - (CH - n_tok);
                    by_token[it] = w.sa * power(lg, (i > 0 ? i : 0) + w.e0) * s_unit;
                }
#pragma unroll
            for (int it = 0; it < NB; it++)
#pragma unroll
                for (int v = 0; v < VB; v++) O[it][v] = (f4)0.f;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                Part pa[NB][P];
#pragma unroll
                for (int it = 0; it < NB; it++) parts_of(pa[it], fa[it][f]);
#pragma unroll
                for (int v = 0; v < VB; v++) {
                    Part fs[TWO];
                    float y[FE];
#pragma unroll
                    for (int e = 0; e < FE; e++) {
                        int i = f * FE + e, u = HALF ? i / 4 : i % VA, r = HALF ? i % 4 : i / VA;
                        y[e] = S[u][v][r];
                    }
                    split(fs, y);
#pragma unroll
                    for (int it = 0; it < NB; it++) O[it][v] = dots(O[it][v], fs, pa[it]);
                }
            }
#pragma unroll
            for (int v = 0; v < VB; v++) {
                Part pc[P];
                parts_of(pc, fct[v]);
#pragma unroll
                for (int it = 0; it < NB; it++) {
                    O[it][v] *= by_token[it];
                    if (inside && from[it]) O[it][v] = (f4)0.f;
                    O[it][v] = dots(O[it][v], pc, fp[it]);
                }
            }
        }

        // the state: c weighted by its decay to the chunk's end.  In 16 bits the weighted value goes in as two parts (2^-16, enough
        // for o), and as three where the state itself is an answer, in float32 (bf16, 500 x 1024 x 4 heads of 64: forward 270 us with
        // two, 271 with three, forward and backward 855 and 880).  S is touched only where the unit has become small.
        float keep = n_tok < CH ? power(lg, n_tok) : whole, unit_new = s_unit * keep;
        const bool off = unit_new < 1.f / 65536 || inside;
        unit_new = off ? 1.f : unit_new;
        if (__builtin_amdgcn_readfirstlane(off)) {
            keep *= s_unit * __builtin_amdgcn_rcpf(unit_new);
#pragma unroll
            for (int u = 0; u < VA; u++)
#pragma unroll
                for (int v = 0; v < VB; v++) S[u][v] = inside ? (f4)0.f : S[u][v] * keep;
        }
        if (inside) any = 1;
        s_unit = unit_new;
        const float grow = __builtin_amdgcn_rcpf(unit_new);
        float by[FE];
#pragma unroll
        for (int e = 0; e < FE; e++) by[e] = !inside || e / 4 * 16 + e % 4 + 4 * g >= last ? enter[e] * grow : 0.f;
#pragma unroll
        for (int v = 0; v < VB; v++) {
            Part y[TWO], rest[1];
            float z[FE];
#pragma unroll
            for (int e = 0; e < FE; e++) z[e] = rounded((float)fct[v][e] * by[e]);
            split(y, z);
#pragma unroll
            for (int u = 0; u < VA; u++) {
                Part pb[P];
                parts_of(pb, fbt[u]);
                S[u][v] = dots(S[u][v], pb, y);
            }
            if (HALF && w.answer) {
                split(rest, z);
#pragma unroll
                for (int u = 0; u < VA; u++) {
                    Part pb[P];
                    parts_of(pb, fbt[u]);
                    S[u][v] = dot(S[u][v], pb[0], rest[0]);
                    if (P == 2) S[u][v] = dot(S[u][v], pb[P - 1], y[TWO - 1]);
                }
            }
        }
        done();
        if constexpr (!STATE) {
#pragma unroll
            for (int it = 0; it < NB; it++)
                if (16 * it + c >= CH - n_tok) {
                    T* to = po + (int64_t)(x + 16 * it - (CH - n_tok)) * sto;
                    constexpr int RUN = HALF ? 8 : 4 * VB;  // neighbouring columns
#pragma unroll
                    for (int q = 0; q < 4 * VB / RUN; q++) {
                        int left = db - j0 - RUN * g - 32 * q;
                        constexpr int N = 16 / sizeof(T);
#pragma unroll
                        for (int e = 0; e < RUN; e += N) {
                            Piece<T, N> y;
#pragma unroll
                            for (int i = 0; i < N; i++) {
                                int v = HALF ? 2 * q + (e + i) / 4 : (e + i) % VB, r = HALF ? (e + i) % 4 : (e + i) / VB;
                                y.v[i] = (T)O[it][v][r];
                            }
                            if (e + N <= left) {
                                *(Piece<T, N>*)(to + 32 * q + e) = y;
                            } else {
#pragma unroll
                                for (int i = 0; i < N; i++)
                                    if (e + i < left) to[32 * q + e + i] = y.v[i];
                            }
                        }
                    }
                }
        }
        return true;
    };

    if (da < L::DA || db - j0 < 16 * VB)
        for (int i = lane * 16; i < L::BUF; i += 1024) *(u4*)(lds + i) = (u4)0u;
    bool fresh;
    unsigned inside;
    int n_tok = chunk(0, &fresh, &inside);
    issue(0, n_tok);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        int d = c - 4 * g - r;
        near[r] = d >= 0 ? w.sa * w.sb * power(lg, d) : 0.f;
        far[r] = w.sa * w.sb * power(lg, 16 + d);
#pragma unroll
        for (int b = 0; b < NB; b++) enter[4 * b + r] = w.sb * power(lg, CH - (16 * b + 4 * g + r) - w.e0);
    }
#pragma unroll
    for (int b = 0; b < NB; b++) carry[b] = w.sa * power(lg, 16 * b + c + w.e0);
    whole = power(lg, CH);
    landed();
    for (int x = 0; x < steps;) {
        const int x_next = x + n_tok;
        bool f_next = false;
        unsigned i_next = 0;
        const int n_next = x_next < steps ? chunk(x_next, &f_next, &i_next) : 0;
        auto begin = [&] {
            if (n_next) issue(x_next, n_next);
        };
        if (!compute(x, n_tok, fresh, inside, begin, landed)) {
            (inside ? cut : slow) = x_next;
            n_tok = chunk(x, &fresh, &inside);
            issue(x, n_tok);
            landed();
            continue;
        }
        x = x_next, n_tok = n_next, fresh = f_next, inside = i_next;
        if (flags && x - seen >= 64) {
            m0 = m1, m1 = __ballot(ahead != 0), seen += 64;
            ahead = flag(seen + 128 + lane);
        }
    }

    if (STATE) {
#pragma unroll
        for (int u = 0; u < VA; u++)
#pragma unroll
            for (int v = 0; v < VB; v++) *held(all, item, VA * VB, u * VB + v, lane) = S[u][v] * s_unit;
        if (lane == 0) all.left[item] = any ? CUT : power(lg, steps);
        return;
    }
    if (!w.s_out || seg + 1 < all.segs) return;
    bool drop = w.s_drop && w.s_drop[n * w.start_sn];
    state_store<L>(S, s_unit, drop, w, w.s_out + (int64_t)nh * da * db, j0, c, g);
}

// The states that the segments begin with, from what each adds: begin_0 = what enters, begin_{s+1} = left_s begin_s + added_s.
// A workgroup takes 32 float4s of one wave's accumulators; its 8 rows of threads take a run of PER segments each, all of whose loads
// are in flight at once, then hand on through LDS (8 heads of 64, 128 segments: 9 us for 34 MB in and out, most of it latency).
constexpr int RUNS = 8, MAX_SEGS = RUNS * 16;

template <class L, int PER>
__global__ __launch_bounds__(256) void k_join(Sweeps all) {
    constexpr int VA = L::VA, VB = L::VB, TILES = VA * VB;
    __shared__ f4 sums[RUNS][32];
    __shared__ float lefts[RUNS];
    unsigned part = blockIdx.x % (2 * TILES), rest = blockIdx.x / (2 * TILES);
    unsigned slice = rest % all.slices, role = rest / all.slices % all.count, nh = rest / all.slices / all.count;
    const Sweep& w = all.w[role];
    if ((int)slice * 16 * VB >= w.db) return;
    const int tile = part / 2, lane = part % 2 * 32 + threadIdx.x % 32, run = threadIdx.x / 32;
    const unsigned s0 = run * PER;
    auto item = [&](unsigned s) { return ((nh * all.segs + s) * all.count + role) * all.slices + slice; };
    f4 add[PER], begin;
    float left[PER];
    int g = lane / 16, c = lane % 16, u = tile / VB, v = tile % VB;
#pragma unroll
    for (int r = 0; r < 4; r++) begin[r] = entering(w, nh, L::dim(u, 4 * g + r), slice * 16 * VB + L::col(v, c));
#pragma unroll
    for (unsigned i = 0; i < PER; i++) {
        bool in = s0 + i < all.segs;
        add[i] = in ? *held(all, item(s0 + i), TILES, tile, lane) : (f4)0.f;
        left[i] = in ? all.left[item(s0 + i)] : 1.f;
    }
    f4 x = (f4)0.f;
    float l = 1.f;
#pragma unroll
    for (int i = 0; i < PER; i++) x = joined(x, left[i], add[i]), l = l == CUT || left[i] == CUT ? CUT : l * left[i];
    sums[run][threadIdx.x % 32] = x;
    if (threadIdx.x % 32 == 0) lefts[run] = l;
    __syncthreads();
    x = begin;
    for (int i = 0; i < run; i++) x = joined(x, lefts[i], sums[i][threadIdx.x % 32]);
#pragma unroll
    for (unsigned i = 0; i < PER; i++)
        if (s0 + i < all.segs) {
            *held(all, item(s0 + i), TILES, tile, lane) = x;
            x = joined(x, left[i], add[i]);
        }
}

constexpr int64_t FILL = 1024;  // waves: one for each SIMD

// Columns of C that a wave holds, by the tile width of a and b and the width of c: as many as its registers take, for they share the
// scores; 64 with tiles of 64 (500 x 1024 x 4 heads of 64, bf16: forward and backward 880 us, 1095 with 32), where c has them and the
// waves fill the chip (with fewer, the time of one wave's chunk counts).
static int columns_of(int tile, int db, int64_t waves) { return tile == 64 && db > 32 && waves >= FILL ? 64 : 32; }

template <typename T, class L>
static void launch_tile(const Sweeps& s, hipStream_t st) {
    unsigned grid = (s.items + 7) / 8 * 8;
    if constexpr (L::VB == 2)  // (64 columns are held where the waves fill the chip: in one segment)
        if (s.segs > 1) {
            k_sweep<T, L, true><<<grid, 64, 0, st>>>(s);
            unsigned parts = s.items / s.segs * L::VA * L::VB * 2;
            if (s.segs > 4 * RUNS) k_join<L, 16><<<parts, 256, 0, st>>>(s);
            else if (s.segs > OWN_JOIN) k_join<L, 4><<<parts, 256, 0, st>>>(s);
        }
    k_sweep<T, L, false><<<grid, 64, 0, st>>>(s);
}

template <typename T>
static void launch(const Sweeps& s, hipStream_t st) {
    if (s.tile == 32) launch_tile<T, Tile<T, 32, 2>>(s, st);
    else if (s.tile == 64 && s.columns == 64) launch_tile<T, Tile<T, 64, 4>>(s, st);
    else if (s.tile == 64) launch_tile<T, Tile<T, 64, 2>>(s, st);
    else launch_tile<T, Tile<T, 128, 2>>(s, st);
}

static int tile(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

// The launch of `count` sweeps, of the widest one's tile.  With fewer waves than fill the chip twice over (one a SIMD is
// half of that) the axis is cut into segments, at least 32 steps each: their states are computed first, then joined.  That costs a
// pass, so fewer than 3 segments or 128 steps stay whole (forward, 4 heads of 32, 500 steps, float32: 24 us with 64 steps or more a
// segment, 20 with 32; 400 heads of 64, 300 steps, bf16: 41 us in 2 segments, 33.5 whole).
static Sweeps plan(const urgym_ops_seq* q, const Sweep* w, int count) {
    Sweeps s = {};
    s.count = count, s.heads = q->heads, s.steps = q->steps, s.log_decay = q->log_decay;
    int db = 0, da = 0;
    for (int i = 0; i < count; i++) s.w[i] = w[i], da = w[i].da > da ? w[i].da : da, db = w[i].db > db ? w[i].db : db;
    s.tile = tile(da), s.columns = columns_of(s.tile, db, q->envs * q->heads * count * ((db + 63) / 64)), s.slices = (db + s.columns - 1) / s.columns;
    s.items = (unsigned)(q->envs * q->heads) * s.count * s.slices;
    int64_t segs = s.items >= FILL ? 1 : 2 * FILL / s.items, most = q->steps / 32;
    segs = segs < most ? segs : most;
    segs = segs < MAX_SEGS ? segs : MAX_SEGS;
    if (segs < 3 || most < 4) segs = 1;
    int64_t len = (q->steps + segs - 1) / segs;
    len = (len + 31) / 32 * 32;
    s.segs = (unsigned)((q->steps + len - 1) / len), s.seg_len = (int)len;
    s.items *= s.segs;
    return s;
}

// in floats, whole vectors
static int64_t workspace(const Sweeps& s) { return s.segs > 1 ? ((int64_t)s.items * (s.tile * s.columns + 1) + 3) / 4 * 4 : 0; }

static void launch(const urgym_ops_seq* q, Sweeps s, float* ws, hipStream_t st) {
    s.ws = ws, s.left = ws + (int64_t)s.items * s.tile * s.columns;
    if (q->dtype == URGYM_OPS_F32) launch<float>(s, st);
    else if (q->dtype == URGYM_OPS_BF16) launch<bf16>(s, st);
    else launch<f16>(s, st);
}

// One token: W waves of a workgroup take one (env, head).  LPR lanes hold a row of the state, E elements each (neighbours, as one
// vector, or LPR apart where dv is odd), and 64 / LPR rows are under way at once in each wave, 8 times over: the state's bytes, in and
// out, are the whole cost (4096 x 4 heads of 64: 99 us, 5.4 TB/s).  The columns' sums over the rows are joined across lanes, then through LDS across the waves.
template <typename T, int E, bool VEC, int LPR>
__global__ __launch_bounds__(256) void k_step(int heads, int dk, int dv, Rows q, Rows k, Rows v, const float* log_decay,
                                              const uint8_t* start, int64_t start_sn, float scale, const float* s_in,
                                              float* s_out, T* o) {
    constexpr int RPP = UO_WAVE / LPR, U = 8;
    typedef float V __attribute__((ext_vector_type(VEC ? E : 1)));
    __shared__ float qs[URGYM_OPS_MAX_HEAD_DIM], ks[URGYM_OPS_MAX_HEAD_DIM], sums[4][E * LPR];
    const int64_t n = blockIdx.x / (unsigned)heads;
    const int h = blockIdx.x % (unsigned)heads, waves = blockDim.x / UO_WAVE, wave = threadIdx.x / UO_WAVE, lane = threadIdx.x % UO_WAVE;
    const int c = lane % LPR, r0 = wave * RPP + lane / LPR;
    const bool fresh = start && start[n * start_sn];
    const T *qr = (const T*)q.p + n * q.sn + h * q.sh, *kr = (const T*)k.p + n * k.sn + h * k.sh, *vr = (const T*)v.p + n * v.sn + h * v.sh;
    auto col = [&](int e) { return VEC ? c * E + e : c + e * LPR; };
    const float* in = s_in + (int64_t)blockIdx.x * dk * dv;
    float* out = s_out + (int64_t)blockIdx.x * dk * dv;
    float s[U][E], x[E], acc[E];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            int i = i0 + u * waves * RPP;
#pragma unroll
            for (int e = 0; e < E; e++) s[u][e] = 0.f;
            if (i < dk && !fresh) {
                if (VEC) {
                    if (c * E < dv) {
                        V y = *(const V*)(in + i * dv + c * E);
#pragma unroll
                        for (int e = 0; e < E; e++) s[u][e] = y[VEC ? e : 0];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if (col(e) < dv) s[u][e] = in[i * dv + col(e)];
                }
            }
        }
    };
    load(r0);
    const float g = power(log_decay[h] * 1.44269504088896340736f, 1);
    for (int i = threadIdx.x; i < dk; i += blockDim.x) qs[i] = scale * (float)qr[i], ks[i] = (float)kr[i];
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = col(e) < dv ? (float)vr[col(e)] : 0.f, acc[e] = 0.f;
    __syncthreads();
    for (int i0 = r0; i0 - r0 < dk; i0 += U * waves * RPP) {
        if (i0 != r0) load(i0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            int i = i0 + u * waves * RPP;
            if (i < dk) {
                float b = ks[i], a = qs[i];
                V y;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    s[u][e] = (fresh ? 0.f : g * s[u][e]) + b * x[e];
                    acc[e] += s[u][e] * a;
                    if (VEC) y[VEC ? e : 0] = s[u][e];
                    else if (col(e) < dv) out[i * dv + col(e)] = s[u][e];
                }
                if (VEC && c * E < dv) *(V*)(out + i * dv + c * E) = y;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
#pragma unroll
        for (int m = LPR; m < UO_WAVE; m *= 2) acc[e] += __shfl_xor(acc[e], m);
        if (waves > 1 && lane < LPR) sums[wave][e * LPR + c] = acc[e];
    }
    if (waves > 1) {
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int e = 0; e < E; e++)
            for (int i = 1; i < waves; i++) acc[e] += sums[i][e * LPR + c];
    }
    if (lane < LPR)
#pragma unroll
        for (int e = 0; e < E; e++)
            if (col(e) < dv) o[(int64_t)blockIdx.x * dv + col(e)] = (T)acc[e];
}

template <typename T>
static void step(int64_t envs, int heads, int dk, int dv, Rows q, Rows k, Rows v, const float* log_decay, const uint8_t* start,
                 int64_t start_sn, float scale, const float* s_in, float* s_out, T* o, hipStream_t st) {
    unsigned grid = (unsigned)(envs * heads);
    bool vec = dv % 4 == 0 && (uintptr_t)s_in % 16 == 0 && (uintptr_t)s_out % 16 == 0;
    int lanes = vec ? dv / 4 : dv, lpr = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
    int rounds = (dk * lpr + UO_WAVE - 1) / UO_WAVE;  // loads of one wave, 8 of which it has under way
    unsigned block = rounds <= 8 ? 64 : rounds <= 16 ? 128 : 256;
#define STEP(E, VEC, LPR) k_step<T, E, VEC, LPR><<<grid, block, 0, st>>>(heads, dk, dv, q, k, v, log_decay, start, start_sn, scale, s_in, s_out, o)
    if (vec) lpr == 8 ? STEP(4, true, 8) : lpr == 16 ? STEP(4, true, 16) : STEP(4, true, 32);
    else if (dv > 64) STEP(2, false, 64);
    else lpr <= 16 ? STEP(1, false, 16) : lpr == 32 ? STEP(1, false, 32) : STEP(1, false, 64);
#undef STEP
}

static int seq_check(const char* what, int dtype, int64_t steps, int64_t envs, int heads, int dk, int dv) {
    if (dtype < 0 || dtype > 2) return uo_fail("%s: unknown dtype %d", what, dtype);
    if (dk < 1 || dk > URGYM_OPS_MAX_HEAD_DIM || dv < 1 || dv > URGYM_OPS_MAX_HEAD_DIM)
        return uo_fail("%s: dk %d and dv %d must be 1 .. %d", what, dk, dv, URGYM_OPS_MAX_HEAD_DIM);
    if (steps < 1 || envs < 1 || heads < 1) return uo_fail("%s: steps %lld, envs %lld, heads %d", what, (long long)steps, (long long)envs, heads);
    if (envs > URGYM_OPS_MAX_HEADS || (int64_t)heads * envs > URGYM_OPS_MAX_HEADS || steps > (1 << 30))
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
    w.s_in = s->state, w.s_i = transposed ? 1 : db, w.s_j = transposed ? da : 1, w.answer = !transposed;
    w.sa = s->scale, w.sb = 1.f, w.e0 = 1;
    return w;
}

// dk or dv: against time's order from d_state_out.  Token x of the sweep is step steps - 1 - x, which an episode border cuts from
// token x - 1 where step steps - x starts one.
static Sweep backward(const urgym_ops_seq* s, Rows a, Rows b, Rows c, Rows o, int da, int db, bool transposed, const float* d_state_out) {
    Sweep w = forward(s, reversed(a, s), reversed(b, s), reversed(c, s), reversed(o, s), da, db, transposed);
    if (s->start) w.start = s->start + s->steps * s->start_stride[0], w.start_st = -s->start_stride[0];
    w.first = false, w.e0 = 0, w.s_in = d_state_out, w.s_drop = s->start;
    w.sa = 1.f, w.sb = s->scale;
    return w;
}

// whether a chunk of rows that lie `st` elements apart is too long for the sweeps' 32-bit offsets
static bool far(int64_t st, int size) { return (st < 0 ? -st : st) >= ((int64_t)1 << 31) / (32 * size); }

// what the sweeps read of r: itself, or (padded rows, appended to the workspace at `floats`) its copy
static Rows readable(const urgym_ops_seq* s, Rows r, int d, float* ws, int64_t* floats, Packs* p) {
    int size = s->dtype == URGYM_OPS_F32 ? 4 : 2, n = 16 / size, width = (d + n - 1) / n * n;
    if (d % n == 0 && (uintptr_t)r.p % 16 == 0 && r.st % n == 0 && r.sn % n == 0 && r.sh % n == 0 && !far(r.st, size)) return r;
    Rows to = {ws + *floats, s->envs * s->heads * width, (int64_t)s->heads * width, width};
    if (far(to.st, size)) to = {to.p, width, s->heads * s->steps * width, s->steps * width};
    p->t[p->count++] = {r, to, d};
    *floats += s->steps * s->envs * s->heads * width * size / 4;
    return to;
}

// Everything one direction enqueues, and its workspace: copies of what cannot be read as it is, then the launches of o's sweep, or
// of those of dk, dq and dv, which read the same rows and share a launch where their tiles agree or may.
struct Work {
    Packs packs;
    Sweeps sweeps[2];
    int count;
    float* ws;         // of the sweeps
    int64_t floats;    // in all
};

static Work work(const urgym_ops_seq* s, const Rows* g, float* ws) {
    Work w = {};
    w.packs.heads = s->heads, w.packs.envs = (unsigned)s->envs, w.packs.steps = s->steps;
    Rows q = readable(s, rows(s->q, s->q_stride), s->dk, ws, &w.floats, &w.packs), k = readable(s, rows(s->k, s->k_stride), s->dk, ws, &w.floats, &w.packs),
         v = readable(s, rows(s->v, s->v_stride), s->dv, ws, &w.floats, &w.packs);
    Rows none = {};
    if (!g) {
        Sweep o = forward(s, q, k, v, none, s->dk, s->dv, false);
        w.sweeps[w.count++] = plan(s, &o, 1);
    } else {
        Rows d = readable(s, *g, s->dv, ws, &w.floats, &w.packs);
        Sweep b[3] = {backward(s, v, d, q, none, s->dv, s->dk, true, nullptr), forward(s, d, v, k, none, s->dv, s->dk, true),
                      backward(s, k, q, d, none, s->dk, s->dv, false, nullptr)};
        // Tiles of 32 and 64 in 16 bits share the wider one where waves are few and launches count (24 and 40 wide heads, 333 steps, forward
        // and backward, bf16 and float16: 185 heads 81 -> 69 and 91 -> 85 us, 370 heads 105 -> 99 and 119 either way, but 740 heads 127 ->
        // 142 and 151 -> 171); wider ones lose sooner (64 and 128 wide, bf16: 45 heads 80 -> 70, but 185 heads
        // 117 -> 136, 370 heads 146 -> 188).
        bool few = s->dtype != URGYM_OPS_F32 && s->dk <= 64 && s->dv <= 64 && s->envs * s->heads < FILL / 2;
        if (tile(s->dk) == tile(s->dv) || few) w.sweeps[w.count++] = plan(s, b, 3);
        else w.sweeps[w.count++] = plan(s, b, 2), w.sweeps[w.count++] = plan(s, b + 2, 1);
    }
    w.ws = ws + w.floats;
    int64_t most = 0;
    for (int i = 0; i < w.count; i++) most = workspace(w.sweeps[i]) > most ? workspace(w.sweeps[i]) : most;
    w.floats += most;
    return w;
}

extern "C" int64_t urgym_ops_decay_workspace(const urgym_ops_seq* s) {
    if (seq_check("urgym_ops_decay_workspace", s)) return -1;
    return work(s, nullptr, nullptr).floats;
}

extern "C" int64_t urgym_ops_decay_backward_workspace(const urgym_ops_seq* s, const void* d_out, const int64_t d_out_stride[3]) {
    if (seq_check("urgym_ops_decay_backward_workspace", s)) return -1;
    if (!d_out_stride) return uo_fail("urgym_ops_decay_backward_workspace: d_out's strides are needed");
    Rows g = rows(d_out, d_out_stride);
    return work(s, &g, nullptr).floats;
}

static int run(const char* what, const urgym_ops_seq* s, const Work& w, hipStream_t st) {
    if (w.packs.count) {
        int size = s->dtype == URGYM_OPS_F32 ? 4 : 2, n = 16 / size;
        int64_t pieces = (int64_t)s->envs * s->heads * (((s->dk > s->dv ? s->dk : s->dv) + n - 1) / n);
        dim3 grid((unsigned)((pieces + 255) / 256), (unsigned)(s->steps < 65535 ? s->steps : 65535), w.packs.count);
        if (s->dtype == URGYM_OPS_F32) k_pack<float><<<grid, 256, 0, st>>>(w.packs);
        else k_pack<f16><<<grid, 256, 0, st>>>(w.packs);
    }
    for (int i = 0; i < w.count; i++) launch(s, w.sweeps[i], w.ws, st);
    return uo_launched(what);
}

extern "C" int urgym_ops_decay(const urgym_ops_seq* s, void* o, float* state_out, float* ws, void* stream) {
    if (seq_check("urgym_ops_decay", s)) return -1;
    if (!o || !state_out) return uo_fail("urgym_ops_decay: o and state_out are needed");
    Work w = work(s, nullptr, ws);
    if (w.floats && (!ws || (uintptr_t)ws % 16)) return uo_fail("urgym_ops_decay: a workspace is needed, 16-byte aligned");
    w.sweeps[0].w[0].o = packed(o, s, s->dv), w.sweeps[0].w[0].s_out = state_out;
    return run("urgym_ops_decay", s, w, (hipStream_t)stream);
}

extern "C" int urgym_ops_decay_backward(const urgym_ops_seq* s, const void* d_out, const int64_t d_out_stride[3],
                                        const float* d_state_out, void* dq, void* dk, void* dv, float* d_state, float* ws,
                                        void* stream) {
    if (seq_check("urgym_ops_decay_backward", s)) return -1;
    if (!d_out || !d_out_stride || !dq || !dk || !dv) return uo_fail("urgym_ops_decay_backward: d_out, dq, dk and dv are needed");
    Rows g = rows(d_out, d_out_stride);
    Work w = work(s, &g, ws);
    if (w.floats && (!ws || (uintptr_t)ws % 16)) return uo_fail("urgym_ops_decay_backward: a workspace is needed, 16-byte aligned");
    Sweep &k = w.sweeps[0].w[0], &q = w.sweeps[0].w[1], &v = w.count == 1 ? w.sweeps[0].w[2] : w.sweeps[1].w[0];
    k.o = reversed(packed(dk, s, s->dk), s), q.o = packed(dq, s, s->dk), v.o = reversed(packed(dv, s, s->dv), s);
    k.s_in = v.s_in = d_state_out, v.s_out = d_state;
    return run("urgym_ops_decay_backward", s, w, (hipStream_t)stream);
}

extern "C" int urgym_ops_decay_step(int dtype, int64_t envs, int heads, int dk, int dv, const void* q, int64_t q_sn, int64_t q_sh,
                                    const void* k, int64_t k_sn, int64_t k_sh, const void* v, int64_t v_sn, int64_t v_sh,
                                    const float* log_decay, const uint8_t* start, int64_t start_stride, float scale,
                                    const float* state, float* state_out, void* o, void* stream) {
    if (seq_check("urgym_ops_decay_step", dtype, 1, envs, heads, dk, dv)) return -1;
    if (!q || !k || !v || !log_decay || !state || !state_out || !o) return uo_fail("urgym_ops_decay_step: a pointer is missing");
    Rows rq = {q, 0, q_sn, q_sh}, rk = {k, 0, k_sn, k_sh}, rv = {v, 0, v_sn, v_sh};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == URGYM_OPS_F32) step(envs, heads, dk, dv, rq, rk, rv, log_decay, start, start_stride, scale, state, state_out, (float*)o, st);
    else if (dtype == URGYM_OPS_BF16) step(envs, heads, dk, dv, rq, rk, rv, log_decay, start, start_stride, scale, state, state_out, (bf16*)o, st);
    else step(envs, heads, dk, dv, rq, rk, rv, log_decay, start, start_stride, scale, state, state_out, (f16*)o, st);
    return uo_launched("urgym_ops_decay_step");
}
