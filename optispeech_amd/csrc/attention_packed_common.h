// Shared by the translation units of attention over documents (attention_packed_fwd.hip, attention_packed_bwd.hip, attention_packed_token.hip):
// arguments, operand tiles, the two matrix products and the score function.
//
//   x = scale q_i . k_j;   c = cap tanh(x / cap) (cap > 0, else x);   s = c - slope_h |pos_i - j|;   pos_i = keys - queries + i
//   query i sees the keys j < lim_i:   full: all;   causal: lim_i = max(pos_i + 1, prefix)   (a causal and a prefix mask are one limit)
//   o_i = sum_j softmax_j(s) v_j over the seen keys, 0 where none is seen;  query head h reads key head h / (Hq / Hk)
//
// Scores are kept in units of log2 (everything is multiplied by log2 e), so that a probability is one v_exp_f32.
//
// Matrix layouts, 32 x 32 tiles (l31 = lane & 31, half = lane >> 5): an A operand holds row l31, a B operand column l31; accumulator element i of a
// lane is row (i >> 2) * 8 + 4 half + (i & 3), column l31.  bf16: k = 16 a step, a lane holds k = 8 half .. + 7 (v_mfma_f32_32x32x16_bf16);
// f32: k = 2 a step, a lane holds k = half (v_mfma_f32_32x32x2_f32).
//   score product  X (32 rows x 32 columns) = R C^T: R's rows from LDS (A), C's rows in registers (B): a lane owns one column entity.
//   value product  Y^T (width x columns) += W^T X: X's accumulators ARE the B operand when the k indices of a step are taken in accumulator
//     order; W^T (A) is read from W's LDS rows, bf16 with the transposing ds_read_b64_tr_b16.  The result is transposed: a lane still owns its
//     column entity, so a softmax's rescaling is one factor per lane and needs no exchange.
#pragma once
#include "packed_common.h"

namespace pattn {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float EMPTY = 1.0e30f;             // log-sum-exp of a query that sees nothing: exp2(s - EMPTY) = 0
constexpr float NONE = -1.0e30f;             // running maximum before the first seen key

enum { CAP = 1, SLOPE = 2, WIDE = 4 };       // score function of an instantiation; WIDE (with CAP, bf16 tensors): a cap above WIDE_CAP
constexpr float WIDE_CAP = 512.f;

struct Args {
    const void *q, *k, *v, *o, *dout;
    void* rest;                                         // bf16: o's rounding error, (rows, heads, D), or null
    int64_t qr, qh, kr, kh, vr, vh, dor, doh;           // row and head strides in elements (o and the gradients: (rows, heads, D) contiguous)
    void *out, *dq, *dk, *dv;
    float *lse, *delta;                                 // (Hq, Mq): log2-sum-exp, sum_d dO O
    const int64_t *qbegin, *qlen, *kbegin, *klen;       // per document
    const PackedTile* tiles;
    const int* ntiles;
    const int64_t* prefix;                              // per document or null
    const float* slopes;                                // per query head or null
    int64_t Mq, Mk, docs, qlongest, klongest;           // the last two: the host's bounds on a document, used to choose a kernel only
    float* partial;                                     // dK, dV of the parts of a key head's query heads: (2, parts, Mk, Hk, D)
    int64_t part_size;
    int cap_tiles, Hq, Hk, G, D, causal, parts;
    float scale, softcap;
};

template <typename T> struct Op;

template <> struct Op<__bf16> {
    typedef pk_bf16x8 Frag;
    static constexpr int EPC = 8;                                        // elements of a 16-byte chunk
    template <int DP> static constexpr int NF = DP / 16;
    static __device__ __forceinline__ f32x16 mma(const Frag a, const Frag b, const f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    // X as the B operand of a value product: 2 steps of 16 rows
    struct Cols { Frag f[2]; };
    static __device__ __forceinline__ void set(Cols& x, int i, float p) { x.f[i >> 3][i & 7] = (__bf16)p; }   // probabilities enter the matrix pipe as bf16
    static __device__ __forceinline__ float get(const Cols& x, int i) { return (float)x.f[i >> 3][i & 7]; }
    // Which channels a result block holds: rows 0 .. 15 of block d are the channels 16 d .., rows 16 .. 31 the channels DP / 2 + 16 d .. : the four
    // 16-lane groups of a transposing read then touch different banks (rows are one chunk apart, the two column groups half a row): 2 instead of
    // 6 conflict cycles a read.
    template <int DP> static __device__ __forceinline__ int channel(int d, int g4, int half) { return 16 * d + (g4 >> 1) * (DP / 2) + (g4 & 1) * 8 + 4 * half; }
    template <int DP> static __device__ __forceinline__ void value(f32x16 (&y)[DP / 32], const Cols& x, const char* w_l, int lane) {
        constexpr int ROW = DP * 2 + 16;
        const int half = lane >> 5, r16 = lane & 15, g16 = (lane >> 4) & 1;
        const char* base = w_l + (4 * half + (r16 >> 2)) * ROW + (DP / 2 * g16 + 4 * (r16 & 3)) * 2;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) {
                union { s16x4 h[2]; Frag f; } u;
                const char* a = base + 16 * s * ROW + d * 32;
                u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a));
                u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 8 * ROW));
                y[d] = mma(u.f, x.f[s], y[d]);
            }
    }
    template <int DP> static __device__ __forceinline__ f32x16 score(const char* rows_l, const Frag (&c)[DP / 16], int l31, int half, f32x16 acc) {
        constexpr int ROW = DP * 2 + 16;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) acc = mma(*reinterpret_cast<const Frag*>(rows_l + l31 * ROW + (16 * s + 8 * half) * 2), c[s], acc);
        return acc;
    }
    // the same with C's rows in LDS too
    template <int DP> static __device__ __forceinline__ f32x16 score_lds(const char* rows_l, const char* c_l, int l31, int half, f32x16 acc) {
        constexpr int ROW = DP * 2 + 16;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const int at = l31 * ROW + (16 * s + 8 * half) * 2;
            acc = mma(*reinterpret_cast<const Frag*>(rows_l + at), *reinterpret_cast<const Frag*>(c_l + at), acc);
        }
        return acc;
    }
};

template <> struct Op<float> {
    typedef f32x4 Frag;                                                  // 4 steps: k = (8 g + e, 8 g + 4 + e)
    static constexpr int EPC = 4;
    template <int DP> static constexpr int NF = DP / 8;
    static __device__ __forceinline__ f32x16 mma(float a, float b, const f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
    struct Cols { f32x16 f; };
    static __device__ __forceinline__ void set(Cols& x, int i, float p) { x.f[i] = p; }
    static __device__ __forceinline__ float get(const Cols& x, int i) { return x.f[i]; }
    template <int DP> static __device__ __forceinline__ int channel(int d, int g4, int half) { return 32 * d + g4 * 8 + 4 * half; }
    template <int DP> static __device__ __forceinline__ void value(f32x16 (&y)[DP / 32], const Cols& x, const char* w_l, int lane) {
        constexpr int ROW = DP * 4 + 16;
        const int half = lane >> 5, l31 = lane & 31;
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
                y[d] = mma(*reinterpret_cast<const float*>(w_l + ((i >> 2) * 8 + 4 * half + (i & 3)) * ROW + (d * 32 + l31) * 4), x.f[i], y[d]);
    }
    template <int DP> static __device__ __forceinline__ f32x16 score(const char* rows_l, const Frag (&c)[DP / 8], int l31, int half, f32x16 acc) {
        constexpr int ROW = DP * 4 + 16;
#pragma unroll
        for (int g = 0; g < DP / 8; ++g) {
            const Frag r = *reinterpret_cast<const Frag*>(rows_l + l31 * ROW + (8 * g + 4 * half) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = mma(r[e], c[g][e], acc);
        }
        return acc;
    }
};

// Up to R rows of one head behind a buffer descriptor: what lies behind the last valid row or behind channel D reads as zeros, without a branch.
// (Offsets inside a tile stay below 2^31: at most 128 rows of less than 2^24 bytes, checked on the host.)
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const T* base, int64_t row_stride, int rows) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
    const int bytes = __builtin_amdgcn_readfirstlane(max(rows, 0) * (int)(row_stride * (int64_t)sizeof(T)));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), 0, bytes, 0x00020000);
}
constexpr int OUT = (int)0x80000000;         // an offset no descriptor reaches
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 buffer_chunk(__amdgpu_buffer_rsrc_t b, int offset) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 0));
}

// register fragments (B operand of a score product) of row `row` of a buffer
template <typename T, int DP>
__device__ __forceinline__ void load_frags(typename Op<T>::Frag (&f)[Op<T>::template NF<DP>], __amdgpu_buffer_rsrc_t b, int64_t row_stride, int row, int D, int half) {
    typedef typename Op<T>::Frag Frag;
    constexpr int E = Op<T>::EPC;
    const int at = row * (int)(row_stride * (int64_t)sizeof(T));
#pragma unroll
    for (int s = 0; s < Op<T>::template NF<DP>; ++s) {
        const int d = (2 * s + half) * E;
        f[s] = __builtin_bit_cast(Frag, buffer_chunk(b, d < D ? at + d * (int)sizeof(T) : OUT));
    }
}

// Fragments that a loop reads are waited for in front of it: a wait left to their first use would stand in the loop and, from the second turn on, wait
// for the loads that were sent ahead for the next tile.
template <typename F, int N>
__device__ __forceinline__ void settle(F (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// R rows of one head -> LDS in two halves: request into registers, store later.  Row stride in LDS: DP elements and 16 bytes (a shift of four banks
// from row to row).  Rows from `rows` on and channels from D on are zeros: what lies behind a document never enters a product.
template <typename T, int DP, int R, int NT>
struct Stage {
    static constexpr int E = Op<T>::EPC, CPR = DP / E, CHUNKS = R * CPR, N = (CHUNKS + NT - 1) / NT;
    static constexpr bool EVEN = NT % CPR == 0;                          // a thread's chunks lie NT / CPR rows apart: one offset and a step
    f32x4 x[N];
    int off[EVEN ? 1 : N], step;
    __device__ __forceinline__ Stage(int64_t row_stride, int D, int tid) {
        const int rb = (int)(row_stride * (int64_t)sizeof(T));
        step = NT / CPR * rb;
#pragma unroll
        for (int it = 0; it < (EVEN ? 1 : N); ++it) {
            const int i = tid + it * NT, r = i / CPR, c = i - r * CPR;
            off[it] = c * E < D && i < CHUNKS ? r * rb + c * 16 : OUT;   // (OUT and a few steps stay out of reach)
        }
    }
    __device__ __forceinline__ void load(const T* base, int64_t row_stride, int rows) {
        const __amdgpu_buffer_rsrc_t b = row_buffer(base, row_stride, min(rows, R));
#pragma unroll
        for (int it = 0; it < N; ++it) x[it] = buffer_chunk(b, EVEN ? off[0] + it * step : off[EVEN ? 0 : it]);
    }
    __device__ __forceinline__ void store(char* dst, int tid) const {
        constexpr int ROW = DP * (int)sizeof(T) + 16;
#pragma unroll
        for (int it = 0; it < N; ++it) {
            const int i = tid + it * NT, r = i / CPR, c = i - r * CPR;
            if (CHUNKS % NT == 0 || i < CHUNKS) *reinterpret_cast<f32x4*>(dst + r * ROW + c * 16) = x[it];
        }
    }
};

// the values of the same column in both halves of the wave: v_permlane32_swap exchanges the upper half of one register with the lower half of the
// other.  Written in assembly because the builtin hands back its first result twice here; the waits cover a vector write before and a read behind.
__device__ __forceinline__ void half_swap(float v, float& lo, float& hi) {
    lo = v;
    hi = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(lo), "+v"(hi));
}
__device__ __forceinline__ float half_max(float v) { float a, b; half_swap(v, a, b); return fmaxf(a, b); }
__device__ __forceinline__ float half_sum(float v) { float a, b; half_swap(v, a, b); return a + b; }

__device__ __forceinline__ f32x16 splat(float v) {
    f32x16 x;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = v;
    return x;
}

// The score function of a raw product x = q . k (scale > 0), in log2 units, as  s = a u + b:
//   plain: u = x, a = scale log2 e;   cap: u = -1 / (exp(2 y) + 1) with y = scale x / cap, a = 2 cap log2 e, b = cap log2 e  (cap tanh y = cap - 2 cap / (exp
//   2 y + 1) on v_exp_f32 and v_rcp_f32: off by 2^-22 of the cap at most);  EXACT (f32 tensors) and WIDE: u = tanh y by the library, a = cap log2 e, whose
//   error is relative to the score.  WIDE starts at a cap of 512, where the first form is off by 1.2e-4 (a probability's rounding to bf16: 2e-3); on
//   either side of it (caps 512 and 513, causal): 4 x 4096 rows, 16 heads of 128 sharing 4: forward 358 and 430 us, training 1.69 and 2.26 ms;  24 x 700 rows,
//   8 heads of 64: 36 and 50 us, 143 and 192 us;  48 new tokens over 8192 keys each: 92 us both
//   slope: u becomes the score itself with the distance's penalty, a = 1, b = 0
// A maximum over u is a maximum over s, and a u + b - max is one FMA in front of the exponential.
// The cap's derivative 1 - tanh^2 y is 4 (-u - u u) for the first form: the factor 4 goes to the caller (grad_scale).
template <int MODE, bool EXACT>
struct Score {
    static constexpr bool LIB = EXACT || (MODE & WIDE);
    float c1, a, b, fa, fb, slope2;
    __device__ __forceinline__ Score(const Args& p, int head) {
        c1 = 0.f; slope2 = 0.f;
        if constexpr (!(MODE & CAP)) { a = p.scale * LOG2E; b = 0.f; }
        else if constexpr (LIB) { c1 = p.scale / p.softcap; a = p.softcap * LOG2E; b = 0.f; }
        else { c1 = 2.f * p.scale * LOG2E / p.softcap; a = 2.f * p.softcap * LOG2E; b = p.softcap * LOG2E; }
        fa = a; fb = b;
        if constexpr (MODE & SLOPE) { fa = 1.f; fb = 0.f; }
        set_head(p, head);
    }
    __device__ __forceinline__ void set_head(const Args& p, int head) { if constexpr (MODE & SLOPE) slope2 = p.slopes[head] * LOG2E; }
    __device__ __forceinline__ float cap(float x) const {
        if constexpr (!(MODE & CAP)) return x;
        if constexpr (LIB) return tanhf(x * c1);
        return -__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * c1) + 1.f);
    }
    __device__ __forceinline__ float penalise(float u, float distance) const {
        if constexpr (MODE & SLOPE) return fmaf(u, a, fmaf(-slope2, fabsf(distance), b));
        return u;
    }
    // derivative of the capped score by the raw one, from cap(x), without grad_scale
    __device__ __forceinline__ float derive(float c) const { return LIB ? fmaf(-c, c, 1.f) : fmaf(-c, c, -c); }
    static constexpr float grad_scale = (MODE & CAP) && !LIB ? 4.f : 1.f;
};

// host: too few tiles of 128 rows (of `heads` heads) to fill the chip: the waves of a workgroup share 32 rows instead of owning 32 each.  `path`: rows a
// workgroup walks at most (times its heads).  Measured on both sides (causal, forward / dQ + dK + dV, us, wide -> split; n = tiles x heads):
//   f32, width 64:   300 rows n = 90: 28 -> 18 / 95 -> 54, n = 182: 28 -> 29 / 98 -> 95, n = 360: 40 -> 46;  1000 rows n = 264: 86 -> 62 / 287 -> 211;
//                    4000 rows n = 254: 293 -> 186 / 1048 -> 610, n = 1016: 579 -> 636
//   bf16, width 128: 300 rows n = 22: 13.5 -> 10.5 / 38 -> 29, n = 90: 14.3 -> 13.5 / 41 -> 48;  1000 rows n = 66: 30 -> 17 / 89 -> 69, n = 264: 34 -> 35 /
//                    98 -> 133;  4000 rows n = 248: 95 -> 72 / 307 -> 301, n = 1016: 164 -> 266
static inline bool split_waves(int64_t rows, int64_t docs, int64_t heads, int64_t path, bool f32, bool narrow_limit) {
    const int64_t n = (rows / PACKED_TILE + docs / 2) * heads;
    if (f32) return n < (path >= 512 ? 384 : 192);
    if (narrow_limit) return n < 72;                     // gradients of wide bf16 heads: the private tiles cost occupancy
    return n < (path >= 2048 ? 384 : 128);
}

// host: the score function of a call
static inline int score_mode(const Args& p, bool bf16) {
    return (p.softcap > 0.f ? CAP : 0) | (p.slopes ? SLOPE : 0) | (bf16 && p.softcap > WIDE_CAP ? WIDE : 0);
}

// host: a tile's rows fit a buffer descriptor, and a row reaches no further than the next
static inline bool row_stride_ok(int64_t stride, int64_t D, int64_t bf16) { return stride >= D && stride * (bf16 ? 2 : 4) < (int64_t)1 << 24; }

// keys a query at position pos sees
__device__ __forceinline__ int key_limit(int pos, int klen, int prefix, int causal) {
    return causal ? min(max(pos + 1, min(prefix, klen)), klen) : klen;
}

// host: the padded head width an instantiation is made for
static inline int padded_width(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

}  // namespace pattn
