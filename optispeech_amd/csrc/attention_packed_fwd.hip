// Attention over documents, forward: capped scores, a penalty on distance, document, causal and prefix masks, shared key heads.
// Scores and masks: attention_packed_common.h.  For a backward the kernel keeps one number per query and head, the log2-sum-exp of its scores, and for
// bf16 results what their rounding took off (`rest`, bf16): the backward's delta = sum dO O would otherwise carry that rounding into every
// element of a row of dS alike.
//
// One workgroup = 4 waves = one tile of 128 queries of one head; a wave owns 32 queries (one per lane, both halves of the wave hold the same
// query and half of the keys).  Keys and values pass through LDS in tiles (64 rows, f32: 32), two buffers, one barrier per tile: the next tile's
// rows are requested into registers before the current tile is computed and stored to the other buffer behind its products.
//   S^T (keys x queries) = K Q^T;  running maximum and sum per lane;  O^T (width x queries) += V^T P^T
// The running maximum is moved only when a row's maximum grows by more than 8 (a factor of 256 in the probabilities, which f32 sums and bf16
// operands carry without loss): the rescaling of O is skipped for nearly every tile after the first.
//
// Measured (bf16): 24 causal prompts of 1 .. 2048 rows, 8 heads of 64, penalised distances: 65 - 73 us (490 - 540 TFLOP/s);  8 x 4096 rows, 16 heads of 128,
// bidirectional: 1.44 ms, 764 TFLOP/s, the matrix pipe busy half of the cycles at the 1.34 GHz the chip's power allows (a library product of 8192^3: 1193).
// Bound by the issue of two waves a SIMD: 256 cycles of matrix work and 250 (plain) to 600 (capped) of vector work for 32 x 32 scores and a width of 64.
// Tried and dropped: 64 queries a wave, one wave a SIMD (K and V leave LDS once for two blocks): 690 -> 440 TFLOP/s, nothing left to run beside the
// products; eight LDS reads sent ahead of the products: no change, the SIMD's second wave covers them.
#include "attention_packed_common.h"
#include <type_traits>

namespace {
using namespace pattn;

// FINE (for a backward, bf16): a probability enters the value product as two bf16 numbers, p = hi + lo.  With one, o is off by 2^-9 of its largest terms, and
// delta = sum dO O with it: the same amount in every element of a row of dS, which a peaked softmax carries into dQ and dK (error of dQ on 18 k rows with
// capped scores of deviation 4: 2.8e-3 -> 2.4e-3, what rounding dS and dQ alone gives).
template <typename T, int DP, int MODE, bool FINE>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : 2) void packed_attn_fwd_kernel(const Args p) {
    typedef Op<T> O;
    constexpr int KT = sizeof(T) == 2 ? 64 : 32, NB = KT / 32, ROW = DP * (int)sizeof(T) + 16;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) char lds[2][2][KT * ROW];                  // [buffer][K, V]
    const int h = blockIdx.x % p.Hq, ti = blockIdx.x / p.Hq;
    const PackedTile tile = p.tiles[ti];                         // (beside the count: the list has cap_tiles entries, its rest is not used)
    if (ti >= p.ntiles[1]) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, half = lane >> 5;
    const int w0 = wave * 32, qi = w0 + l31;                                           // this lane's query in the tile
    const int64_t qrow = (int64_t)tile.row0 + qi;
    T* out = reinterpret_cast<T*>(p.out) + (qrow * p.Hq + h) * p.D;
    if (tile.doc < 0) {                                                                // rows of no document
        if (qi < tile.n)
            for (int d = half * 8; d < p.D; d += 16)
                for (int e = 0; e < 8; ++e) out[d + e] = (T)0.f;
        return;
    }
    const int qlen = (int)p.qlen[tile.doc], klen = (int)p.klen[tile.doc];
    const int prefix = p.prefix ? (int)min(max(p.prefix[tile.doc], (int64_t)0), (int64_t)klen) : 0;
    const int64_t kb = p.kbegin[tile.doc];
    const int hk = h / p.G;
    const T* kp = reinterpret_cast<const T*>(p.k) + kb * p.kr + (int64_t)hk * p.kh;
    const T* vp = reinterpret_cast<const T*>(p.v) + kb * p.vr + (int64_t)hk * p.vh;
    const int off = klen - qlen + tile.i0;                                             // position of the tile's first query
    const int pos = off + qi, lim = qi < tile.n ? key_limit(pos, klen, prefix, p.causal) : 0;
    const int kmax = max(key_limit(off + tile.n - 1, klen, prefix, p.causal), 0);      // keys any query of the tile sees
    const int wmax = w0 < tile.n ? max(key_limit(off + min(w0 + 31, tile.n - 1), klen, prefix, p.causal), 0) : 0;   // ... of the wave
    const int wmin = key_limit(off + w0, klen, prefix, p.causal);                      // keys every query of the wave sees
    typename O::Frag qf[O::template NF<DP>];
    load_frags<T, DP>(qf, row_buffer(reinterpret_cast<const T*>(p.q) + (int64_t)tile.row0 * p.qr + (int64_t)h * p.qh, p.qr, tile.n), p.qr, qi, p.D, half);
    const Score<MODE, EXACT> sc(p, h);
    f32x16 oacc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[d][i] = 0.f;
    settle(qf);
    float m_run = NONE, l_run = 0.f;
    const int nt = (kmax + KT - 1) / KT;
    Stage<T, DP, KT, 256> ks(p.kr, p.D, tid), vs(p.vr, p.D, tid);
    if (nt > 0) {
        ks.load(kp, p.kr, klen);
        vs.load(vp, p.vr, klen);
        ks.store(lds[0][0], tid);
        vs.store(lds[0][1], tid);
        if (nt > 1) { ks.load(kp + KT * p.kr, p.kr, klen - KT); vs.load(vp + KT * p.vr, p.vr, klen - KT); }
    }
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        const int k0 = t * KT;
        const char *kl = lds[t & 1][0], *vl = lds[t & 1][1];
        if (k0 < wmax) {
            f32x16 st[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) st[b] = O::template score<DP>(kl + b * 32 * ROW, qf, l31, half, splat(0.f));
            float mx = -INFINITY;
            const int left = lim - k0 - 4 * half;                                      // rows of the tile this lane's query sees
            auto elements = [&](auto masked) {
                float at = (float)(pos - k0 - 4 * half);
                if constexpr (MODE & SLOPE) asm volatile("" : "+v"(at));              // keeps a whole tile's penalties from being computed ahead of the branch
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int r = b * 32 + (i >> 2) * 8 + (i & 3);
                        float s = sc.penalise(sc.cap(st[b][i]), at - (float)r);
                        if constexpr (masked) s = r < left ? s : -INFINITY;
                        st[b][i] = s;
                        mx = fmaxf(mx, s);
                    }
            };
            if (k0 + KT > wmin) elements(std::true_type{}); else elements(std::false_type{});   // (where every query sees the whole tile)
            mx = fmaf(half_max(mx), sc.fa, sc.fb);
            if (__any(mx > m_run + 8.f)) {
                const float m_new = fmaxf(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) oacc[d][i] *= alpha;
            }
            const float shift = sc.fb - m_run;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                typename O::Cols pc, lo;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(st[b][i], sc.fa, shift));
                    l_run += e;
                    O::set(pc, i, e);
                    if constexpr (FINE) O::set(lo, i, e - O::get(pc, i));
                }
                O::template value<DP>(oacc, pc, vl + b * 32 * ROW, lane);
                if constexpr (FINE) O::template value<DP>(oacc, lo, vl + b * 32 * ROW, lane);
            }
        }
        if (t + 1 < nt) {
            ks.store(lds[(t + 1) & 1][0], tid);
            vs.store(lds[(t + 1) & 1][1], tid);
            if (t + 2 < nt) { ks.load(kp + (int64_t)(k0 + 2 * KT) * p.kr, p.kr, klen - k0 - 2 * KT); vs.load(vp + (int64_t)(k0 + 2 * KT) * p.vr, p.vr, klen - k0 - 2 * KT); }
        }
        __syncthreads();
    }
    const float total = half_sum(l_run), inv = total > 0.f ? 1.f / total : 0.f;        // nothing seen: zeros
    if (qi >= tile.n) return;
    if (p.lse && half == 0) p.lse[(int64_t)h * p.Mq + qrow] = total > 0.f ? m_run + __log2f(total) : EMPTY;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = O::template channel<DP>(d, g, half);
            const float r[4] = {oacc[d][4 * g] * inv, oacc[d][4 * g + 1] * inv, oacc[d][4 * g + 2] * inv, oacc[d][4 * g + 3] * inv};
            if (c < p.D) {
                PackedVec<T, 4>::store(out + c, r);
                if constexpr (!EXACT) {
                    if (p.rest) {
                        const float e[4] = {r[0] - (float)(T)r[0], r[1] - (float)(T)r[1], r[2] - (float)(T)r[2], r[3] - (float)(T)r[3]};
                        PackedVec<T, 4>::store(reinterpret_cast<T*>(p.rest) + (qrow * p.Hq + h) * p.D + c, e);
                    }
                }
            }
        }
}

// The same for few tiles: a workgroup takes 32 queries of a head and its 4 waves walk the keys in turn, each through its own part of LDS and without
// barriers, and join their maxima, sums and outputs in LDS at the end.  Four times the workgroups, each a quarter as long, for four times the
// passes over K and V (out of L2 at these sizes).
template <typename T, int DP, int MODE, bool FINE>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void packed_attn_fwd_split_kernel(const Args p) {
    typedef Op<T> O;
    constexpr int ROW = DP * (int)sizeof(T) + 16, REGION = 2 * 32 * ROW;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) char lds[4][REGION];                        // per wave: K, V; at the end its output
    __shared__ float ml[4][2][32];
    static_assert(REGION >= 32 * DP * 4, "a wave's output fits its part");
    const int h = blockIdx.x % p.Hq, ti = blockIdx.x / p.Hq / 4, q0 = (blockIdx.x / p.Hq & 3) * 32;
    const PackedTile tile = p.tiles[ti];                         // (beside the count: the list has cap_tiles entries, its rest is not used)
    if (ti >= p.ntiles[1]) return;
    if (q0 >= tile.n) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, half = lane >> 5;
    const int qi = q0 + l31, nq = min(32, tile.n - q0);
    const int64_t row0 = (int64_t)tile.row0 + q0;
    T* out = reinterpret_cast<T*>(p.out) + (row0 * p.Hq + h) * p.D;                    // of the first query
    if (tile.doc < 0) {
        for (int u = tid; u < nq * p.D / 8; u += 256)
            for (int e = 0; e < 8; ++e) out[(int64_t)(u / (p.D / 8)) * p.Hq * p.D + u % (p.D / 8) * 8 + e] = (T)0.f;
        return;
    }
    const int qlen = (int)p.qlen[tile.doc], klen = (int)p.klen[tile.doc];
    const int prefix = p.prefix ? (int)min(max(p.prefix[tile.doc], (int64_t)0), (int64_t)klen) : 0;
    const int64_t kb = p.kbegin[tile.doc];
    const int hk = h / p.G;
    const T* kp = reinterpret_cast<const T*>(p.k) + kb * p.kr + (int64_t)hk * p.kh;
    const T* vp = reinterpret_cast<const T*>(p.v) + kb * p.vr + (int64_t)hk * p.vh;
    char *kl = lds[wave], *vl = lds[wave] + 32 * ROW;
    const int off = klen - qlen + tile.i0;
    const int pos = off + qi, lim = qi < tile.n ? key_limit(pos, klen, prefix, p.causal) : 0;
    const int kmax = max(key_limit(off + q0 + nq - 1, klen, prefix, p.causal), 0);
    typename O::Frag qf[O::template NF<DP>];
    load_frags<T, DP>(qf, row_buffer(reinterpret_cast<const T*>(p.q) + row0 * p.qr + (int64_t)h * p.qh, p.qr, nq), p.qr, l31, p.D, half);
    const Score<MODE, EXACT> sc(p, h);
    f32x16 oacc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) oacc[d] = splat(0.f);
    settle(qf);
    float m_run = NONE, l_run = 0.f;
    Stage<T, DP, 32, 64> ks(p.kr, p.D, lane), vs(p.vr, p.D, lane);
    int k0 = wave * 32;
    if (k0 < kmax) { ks.load(kp + (int64_t)k0 * p.kr, p.kr, klen - k0); vs.load(vp + (int64_t)k0 * p.vr, p.vr, klen - k0); }
    for (; k0 < kmax; k0 += 128) {
        __builtin_amdgcn_wave_barrier();
        ks.store(kl, lane);
        vs.store(vl, lane);
        __builtin_amdgcn_wave_barrier();
        if (k0 + 128 < kmax) {
            ks.load(kp + (int64_t)(k0 + 128) * p.kr, p.kr, klen - k0 - 128);
            vs.load(vp + (int64_t)(k0 + 128) * p.vr, p.vr, klen - k0 - 128);
        }
        f32x16 st = O::template score<DP>(kl, qf, l31, half, splat(0.f));
        const float dist = (float)(pos - k0 - 4 * half);
        const int left = lim - k0 - 4 * half;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = (i >> 2) * 8 + (i & 3);
            const float s = sc.penalise(sc.cap(st[i]), dist - (float)r);
            st[i] = r < left ? s : -INFINITY;
            mx = fmaxf(mx, st[i]);
        }
        mx = fmaf(half_max(mx), sc.fa, sc.fb);
        if (__any(mx > m_run + 8.f)) {
            const float m_new = fmaxf(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) oacc[d][i] *= alpha;
        }
        typename O::Cols pc, lo;
        const float shift = sc.fb - m_run;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(fmaf(st[i], sc.fa, shift));
            l_run += e;
            O::set(pc, i, e);
            if constexpr (FINE) O::set(lo, i, e - O::get(pc, i));
        }
        O::template value<DP>(oacc, pc, vl, lane);
        if constexpr (FINE) O::template value<DP>(oacc, lo, vl, lane);
    }
    l_run = half_sum(l_run);
    if (half == 0) { ml[wave][0][l31] = m_run; ml[wave][1][l31] = l_run; }
    __syncthreads();
    float m = NONE, total = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w][0][l31]);
#pragma unroll
    for (int w = 0; w < 4; ++w) total = fmaf(ml[w][1][l31], __builtin_amdgcn_exp2f(ml[w][0][l31] - m), total);
    const float f = total > 0.f ? __builtin_amdgcn_exp2f(m_run - m) / total : 0.f;     // nothing seen: zeros
    if (p.lse && wave == 0 && half == 0 && qi < tile.n) p.lse[(int64_t)h * p.Mq + row0 + l31] = total > 0.f ? m + __log2f(total) : EMPTY;
    float* mine = reinterpret_cast<float*>(lds[wave]);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(mine + l31 * DP + O::template channel<DP>(d, g, half)) =
                f32x4{oacc[d][4 * g] * f, oacc[d][4 * g + 1] * f, oacc[d][4 * g + 2] * f, oacc[d][4 * g + 3] * f};
    __syncthreads();
    const int quads = p.D / 4;
    for (int u = tid; u < nq * quads; u += 256) {
        const int r = u / quads, c = (u - r * quads) * 4;
        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[w]) + r * DP + c);
            a[0] += x[0]; a[1] += x[1]; a[2] += x[2]; a[3] += x[3];
        }
        const int64_t at = (int64_t)r * p.Hq * p.D + c;
        PackedVec<T, 4>::store(out + at, a);
        if constexpr (!EXACT) {
            if (p.rest) {
                const float e[4] = {a[0] - (float)(T)a[0], a[1] - (float)(T)a[1], a[2] - (float)(T)a[2], a[3] - (float)(T)a[3]};
                PackedVec<T, 4>::store(reinterpret_cast<T*>(p.rest) + (row0 * p.Hq + h) * p.D + at, e);
            }
        }
    }
}

template <typename T, int DP, bool FINE>
void launch(const Args& p, hipStream_t s) {
    const int mode = score_mode(p, sizeof(T) == 2);
    const bool split = split_waves(p.Mq, p.docs, p.Hq, p.klongest, sizeof(T) == 4, false);
    const dim3 grid((unsigned)(p.cap_tiles * p.Hq * (split ? 4 : 1)));
#define L(M_)                                                                                                        \
    if (split) hipLaunchKernelGGL((packed_attn_fwd_split_kernel<T, DP, M_, FINE>), grid, dim3(256), 0, s, p);        \
    else hipLaunchKernelGGL((packed_attn_fwd_kernel<T, DP, M_, FINE>), grid, dim3(256), 0, s, p)
    if constexpr (sizeof(T) == 2) {
        if (mode == (CAP | WIDE)) { L(CAP | WIDE); } else if (mode == (CAP | SLOPE | WIDE)) { L(CAP | SLOPE | WIDE); }
    }
    if (mode == 0) { L(0); } else if (mode == 1) { L(1); } else if (mode == 2) { L(2); } else if (mode == 3) { L(3); }
#undef L
}
template <typename T, bool FINE>
void launch_width(const Args& p, hipStream_t s) {
    switch (padded_width(p.D)) {
        case 32: launch<T, 32, FINE>(p, s); break;
        case 64: launch<T, 64, FINE>(p, s); break;
        case 96: launch<T, 96, FINE>(p, s); break;
        default: launch<T, 128, FINE>(p, s);
    }
}
}  // namespace

extern "C" int osp_packed_attention_fwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v,
                                        int64_t v_row, int64_t v_head, int64_t bf16, void* o, void* rest, float* lse, const int64_t* qlen, const int32_t* qtiles,
                                        const int32_t* qntiles, int64_t qcap, const int64_t* kbegin, const int64_t* klen, const int64_t* prefix,
                                        const float* slopes, int64_t docs, int64_t klongest, int64_t Mq, int64_t Hq, int64_t Hk, int64_t D, float scale, float softcap, int64_t causal,
                                        hipStream_t stream) {
    OSP_CHECK_ARG(q && k && v && o && qlen && qtiles && qntiles && kbegin && klen, "null pointer");
    OSP_CHECK_ARG(Hk > 0 && Hq > 0 && Hq % Hk == 0 && Hq <= 65536, "query heads must be a multiple of the key heads");
    OSP_CHECK_ARG(D > 0 && D <= 128 && D % 8 == 0, "head width must be a multiple of 8, at most 128");
    const int E = bf16 ? 8 : 4;
    OSP_CHECK_ARG(q_row % E == 0 && q_head % E == 0 && k_row % E == 0 && k_head % E == 0 && v_row % E == 0 && v_head % E == 0 && packed_aligned(q, 16) &&
                  packed_aligned(k, 16) && packed_aligned(v, 16) && packed_aligned(o, 16), "rows and heads must start on 16 bytes");
    OSP_CHECK_ARG(qcap > 0 && qcap * Hq < (int64_t)1 << 29 && scale > 0.f && softcap >= 0.f && (causal || !prefix), "bad tile list, cap or mask");
    OSP_CHECK_ARG(row_stride_ok(q_row, D, bf16) && row_stride_ok(k_row, D, bf16) && row_stride_ok(v_row, D, bf16), "row strides must lie between the head width and 2^24 bytes");
    Args p = {};
    p.q = q; p.k = k; p.v = v; p.out = o; p.rest = rest; p.lse = lse;
    p.qr = q_row; p.qh = q_head; p.kr = k_row; p.kh = k_head; p.vr = v_row; p.vh = v_head;
    p.qlen = qlen; p.kbegin = kbegin; p.klen = klen; p.tiles = reinterpret_cast<const PackedTile*>(qtiles); p.ntiles = qntiles;
    p.prefix = prefix; p.slopes = slopes; p.Mq = Mq; p.docs = docs; p.klongest = klongest; p.cap_tiles = (int)qcap; p.Hq = (int)Hq; p.Hk = (int)Hk; p.G = (int)(Hq / Hk); p.D = (int)D;
    p.causal = (int)(causal != 0); p.scale = scale; p.softcap = softcap;
    if (!bf16) launch_width<float, false>(p, stream);
    else if (rest) launch_width<__bf16, true>(p, stream);
    else launch_width<__bf16, false>(p, stream);
    OSP_LAUNCH_CHECK();
    return OSP_OK;
}
