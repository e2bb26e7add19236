// Attention over documents, backward: probabilities are recomputed tile by tile from q, k and the log2-sum-exp of the forward.
//   P = exp2(s - lse),  dP = dO V^T,  delta_i = sum_d dO_id O_id  (= sum_j P dP),  dS = P (dP - delta) (1 - tanh^2)
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO;   dK and dV of a shared key head are summed over its query heads
// Scores and masks: attention_packed_common.h.  Two kernels, no atomics, every sum in one fixed order:
//   dq : a wave owns 32 queries and walks the keys (S^T and dP^T per tile, dQ^T += K^T dS^T);  it also writes delta
//   dkv: a wave owns 32 keys with K and V fragments in registers and walks the queries of every head of its group (S and dP, dV^T += dO^T P,
//        dK^T += Q^T dS): the sum over shared heads stays in its accumulators
// S and dP are computed twice, 7 instead of 5 products per tile pair: the price of combining dQ without atomics or a partial dQ per key tile.
// dK / dV keeps V's 128 rows in LDS: with K's and V's fragments both in registers a SIMD held one wave (6.67 ms, below 3.09 ms).
//
// Measured (bf16, 16 heads of 128 sharing 4, capped scores, 5 documents of 1000 .. 8192 rows under a prefix mask): dQ 1.62 ms (845 TFLOP/s), dK / dV 2.51 ms
// (730 TFLOP/s) and 0.11 ms for the sums over the parts of the heads;  32 utterances of 600 .. 800 rows, 2 heads of 128: 54 and 70 us.  Bound like the forward
// (attention_packed_fwd.hip); the cap costs two transcendentals more per score in each kernel.
#include "attention_packed_common.h"
#include <type_traits>

namespace {
using namespace pattn;

// ------------------------------------------------------------------------------------------------ dQ and delta
// dQ^T += K^T dS^T for one tile of 32 keys;  `left`: rows of the tile (4 half taken off) this lane's query sees
template <typename T, int DP, int MODE, bool MASKED>
__device__ __forceinline__ void dq_block(f32x16 (&acc)[DP / 32], const char* kt, const char* vt, const typename Op<T>::Frag (&qf)[Op<T>::template NF<DP>],
                                         const typename Op<T>::Frag (&dof)[Op<T>::template NF<DP>], const Score<MODE, sizeof(T) == 4>& sc, float delta,
                                         float shift, float dist, int left, int lane) {
    typedef Op<T> O;
    const int l31 = lane & 31, half = lane >> 5;
    const f32x16 st = O::template score<DP>(kt, qf, l31, half, splat(0.f));
    const f32x16 dp = O::template score<DP>(vt, dof, l31, half, splat(-delta));       // dP - delta
    if constexpr (MODE & SLOPE) asm volatile("" : "+v"(dist));                         // keeps a whole tile's penalties from being computed ahead of the branch
    typename O::Cols ds;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = (i >> 2) * 8 + (i & 3);
        const float c = sc.cap(st[i]);
        float d = dp[i];
        if constexpr (MODE & CAP) d *= sc.derive(c);
        d *= __builtin_amdgcn_exp2f(fmaf(sc.penalise(c, dist - (float)r), sc.fa, shift));
        if constexpr (MASKED) d = r < left ? d : 0.f;                                  // the product: a query that sees nothing may hold NaN, in dO too
        O::set(ds, i, d);
    }
    O::template value<DP>(acc, ds, kt, lane);
}

template <typename T, int DP, int MODE>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (DP <= 64 ? 3 : 2) : 1) void packed_attn_dq_kernel(const Args p) {
    typedef Op<T> O;
    constexpr int KT = sizeof(T) == 2 ? 64 : 32, NB = KT / 32, ROW = DP * (int)sizeof(T) + 16;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) char lds[2][2][KT * ROW];
    const int h = blockIdx.x % p.Hq, ti = blockIdx.x / p.Hq;
    const PackedTile tile = p.tiles[ti];                         // (beside the count: the list has cap_tiles entries, its rest is not used)
    if (ti >= p.ntiles[1]) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, half = lane >> 5;
    const int w0 = wave * 32, qi = w0 + l31;
    const int64_t qrow = (int64_t)tile.row0 + qi;
    T* out = reinterpret_cast<T*>(p.dq) + (qrow * p.Hq + h) * p.D;
    if (tile.doc < 0) {
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
    const int off = klen - qlen + tile.i0;
    const int pos = off + qi, lim = qi < tile.n ? key_limit(pos, klen, prefix, p.causal) : 0;
    const int kmax = max(key_limit(off + tile.n - 1, klen, prefix, p.causal), 0);
    const int wmax = w0 < tile.n ? max(key_limit(off + min(w0 + 31, tile.n - 1), klen, prefix, p.causal), 0) : 0;
    const int wmin = key_limit(off + w0, klen, prefix, p.causal);
    const bool on = qi < tile.n;
    typename O::Frag qf[O::template NF<DP>], dof[O::template NF<DP>];
    const int64_t row0 = tile.row0, orow = (int64_t)p.Hq * p.D;
    load_frags<T, DP>(dof, row_buffer(reinterpret_cast<const T*>(p.dout) + row0 * p.dor + (int64_t)h * p.doh, p.dor, tile.n), p.dor, qi, p.D, half);
    float delta = 0.f;
    {
        load_frags<T, DP>(qf, row_buffer(reinterpret_cast<const T*>(p.o) + row0 * orow + h * p.D, orow, tile.n), orow, qi, p.D, half);   // o, then q
#pragma unroll
        for (int s = 0; s < O::template NF<DP>; ++s)
#pragma unroll
            for (int e = 0; e < O::EPC; ++e) delta = fmaf((float)dof[s][e], (float)qf[s][e], delta);
        if constexpr (!EXACT) {                                                         // what o's rounding took off
            load_frags<T, DP>(qf, row_buffer(reinterpret_cast<const T*>(p.rest) + row0 * orow + h * p.D, orow, tile.n), orow, qi, p.D, half);
#pragma unroll
            for (int s = 0; s < O::template NF<DP>; ++s)
#pragma unroll
                for (int e = 0; e < O::EPC; ++e) delta = fmaf((float)dof[s][e], (float)qf[s][e], delta);
        }
        delta = half_sum(delta);
        if (on && half == 0) p.delta[(int64_t)h * p.Mq + qrow] = delta;
    }
    load_frags<T, DP>(qf, row_buffer(reinterpret_cast<const T*>(p.q) + row0 * p.qr + (int64_t)h * p.qh, p.qr, tile.n), p.qr, qi, p.D, half);
    const Score<MODE, EXACT> sc(p, h);
    const float shift = sc.fb - (on ? p.lse[(int64_t)h * p.Mq + qrow] : EMPTY), back = p.scale * sc.grad_scale;
    f32x16 acc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    settle(qf);
    settle(dof);
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
            const float dist = (float)(pos - k0 - 4 * half);
            const int left = lim - k0 - 4 * half;                                      // rows of the tile this lane's query sees
            if (k0 + KT > wmin) {
#pragma unroll
                for (int b = 0; b < NB; ++b) dq_block<T, DP, MODE, true>(acc, kl + b * 32 * ROW, vl + b * 32 * ROW, qf, dof, sc, delta, shift, dist - (float)(b * 32), left - b * 32, lane);
            } else {
#pragma unroll
                for (int b = 0; b < NB; ++b) dq_block<T, DP, MODE, false>(acc, kl + b * 32 * ROW, vl + b * 32 * ROW, qf, dof, sc, delta, shift, dist - (float)(b * 32), left - b * 32, lane);
            }
        }
        if (t + 1 < nt) {
            ks.store(lds[(t + 1) & 1][0], tid);
            vs.store(lds[(t + 1) & 1][1], tid);
            if (t + 2 < nt) { ks.load(kp + (int64_t)(k0 + 2 * KT) * p.kr, p.kr, klen - k0 - 2 * KT); vs.load(vp + (int64_t)(k0 + 2 * KT) * p.vr, p.vr, klen - k0 - 2 * KT); }
        }
        __syncthreads();
    }
    if (!on) return;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = O::template channel<DP>(d, g, half);
            const float r[4] = {acc[d][4 * g] * back, acc[d][4 * g + 1] * back, acc[d][4 * g + 2] * back, acc[d][4 * g + 3] * back};
            if (c < p.D) PackedVec<T, 4>::store(out + c, r);
        }
}

// ------------------------------------------------------------------------------------------------ dK, dV
// dV^T += dO^T P, dK^T += Q^T dS for one tile of 32 query rows;  shift: b - log2-sum-exp and ndelta: -delta of the rows, pos0: position of the first row
template <typename T, int DP, int MODE>
__device__ __forceinline__ void dkv_block(f32x16 (&dk)[DP / 32], f32x16 (&dv)[DP / 32], const char* ql, const char* dl, const float* shift_l, const float* ndelta_l,
                                          const typename Op<T>::Frag (&kf)[Op<T>::template NF<DP>],
                                          const typename Op<T>::Frag (&vf)[sizeof(T) == 2 ? 1 : Op<T>::template NF<DP>], const char* v_rows,
                                          const Score<MODE, sizeof(T) == 4>& sc, int pos0, int key, int prefix, bool masked, int lane) {
    typedef Op<T> O;
    const int l31 = lane & 31, half = lane >> 5;
    f32x16 dp;                                                                          // starts at -delta of its rows
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
        const f32x4 del = *reinterpret_cast<const f32x4*>(ndelta_l + g4 * 8 + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[g4 * 4 + e] = del[e];
    }
    const f32x16 sr = O::template score<DP>(ql, kf, l31, half, splat(0.f));
    if constexpr (sizeof(T) == 2) dp = O::template score_lds<DP>(dl, v_rows, l31, half, dp);
    else dp = O::template score<DP>(dl, vf, l31, half, dp);
    const float dist = (float)(pos0 + 4 * half - key);
    const int row_min = key < prefix ? -0x40000000 : key - pos0 - 4 * half;             // rows (4 half taken off) from here on see the key
    typename O::Cols pc, ds;
    auto elements = [&](auto mask) {
        float at = dist;
        if constexpr (MODE & SLOPE) asm volatile("" : "+v"(at));
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const f32x4 shift = *reinterpret_cast<const f32x4*>(shift_l + g4 * 8 + 4 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = g4 * 4 + e, r = g4 * 8 + e;
                const float c = sc.cap(sr[i]);
                float pr = __builtin_amdgcn_exp2f(fmaf(sc.penalise(c, at + (float)r), sc.fa, shift[e]));
                if constexpr (mask) pr = r >= row_min ? pr : 0.f;
                float d = dp[i];
                if constexpr (MODE & CAP) d *= sc.derive(c);
                O::set(pc, i, pr);
                O::set(ds, i, pr * d);
            }
        }
    };
    if (masked) elements(std::true_type{}); else elements(std::false_type{});
    O::template value<DP>(dv, pc, dl, lane);
    O::template value<DP>(dk, ds, ql, lane);
}

template <typename T, int DP, int MODE>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (DP <= 64 ? 3 : 2) : 1) void packed_attn_dkv_kernel(const Args p) {
    typedef Op<T> O;
    constexpr int QT = 32, ROW = DP * (int)sizeof(T) + 16;
    constexpr bool VLDS = sizeof(T) == 2;                                               // V's rows stay in LDS, K's in registers
    __shared__ __attribute__((aligned(16))) char v_l[VLDS ? PACKED_TILE * ROW : 16];
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) char lds[2][2][QT * ROW];                  // [buffer][Q, dO]
    __shared__ __attribute__((aligned(16))) float stat[2][2][QT];                      // [buffer][b - log2-sum-exp, -delta]
    const int hk = blockIdx.x % p.Hk, part = blockIdx.x / p.Hk % p.parts, ti = blockIdx.x / p.Hk / p.parts;
    const int ndoc = p.ntiles[0];
    if (ti >= p.ntiles[1]) return;
    // under a causal mask the first keys have the most queries: the list from its other end
    const PackedTile tile = p.tiles[p.causal && ti < ndoc ? ndoc - 1 - ti : ti];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, half = lane >> 5;
    const int w0 = wave * 32, ki = w0 + l31;
    const int64_t krow = (int64_t)tile.row0 + ki;
    const bool on = ki < tile.n;
    const int64_t at = (krow * p.Hk + hk) * p.D;
    T* outk = reinterpret_cast<T*>(p.dk) + at;
    T* outv = reinterpret_cast<T*>(p.dv) + at;
    if (tile.doc < 0) {
        if (on && p.parts == 1)
            for (int d = half * 8; d < p.D; d += 16)
                for (int e = 0; e < 8; ++e) { outk[d + e] = (T)0.f; outv[d + e] = (T)0.f; }
        return;
    }
    const int qlen = (int)p.qlen[tile.doc], klen = (int)p.klen[tile.doc];
    const int prefix = p.prefix ? (int)min(max(p.prefix[tile.doc], (int64_t)0), (int64_t)klen) : 0;
    const int64_t qb = p.qbegin[tile.doc];
    const int off = klen - qlen;                                                       // position of the document's first query
    // first query that sees a key of the tile: all see the prefix, key j is seen from position j on
    const int first = !p.causal || tile.i0 < prefix ? 0 : max(tile.i0 - off, 0);
    typename O::Frag kf[O::template NF<DP>], vf[VLDS ? 1 : O::template NF<DP>];
    load_frags<T, DP>(kf, row_buffer(reinterpret_cast<const T*>(p.k) + (int64_t)tile.row0 * p.kr + (int64_t)hk * p.kh, p.kr, tile.n), p.kr, ki, p.D, half);
    const T* vrows = reinterpret_cast<const T*>(p.v) + (int64_t)tile.row0 * p.vr + (int64_t)hk * p.vh;
    if constexpr (VLDS) {
        Stage<T, DP, PACKED_TILE, 256> vs(p.vr, p.D, tid);
        vs.load(vrows, p.vr, tile.n);
        vs.store(v_l, tid);
    } else load_frags<T, DP>(vf, row_buffer(vrows, p.vr, tile.n), p.vr, ki, p.D, half);
    settle(kf);
    if constexpr (!VLDS) settle(vf);
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) { dk[d][i] = 0.f; dv[d][i] = 0.f; }
    const int key = tile.i0 + ki;                                                      // this lane's key in the document
    const int nqt = first < qlen ? (qlen - first + QT - 1) / QT : 0, nt = nqt * (p.G / p.parts);
    const int h0 = hk * p.G + part * (p.G / p.parts);                                  // the first of this workgroup's heads
    Score<MODE, EXACT> sc(p, h0);
    const float back = p.scale * sc.grad_scale;
    Stage<T, DP, QT, 256> qs(p.qr, p.D, tid), dos(p.dor, p.D, tid);
    float st_reg = 0.f;
    auto load = [&](int t) {
        const int h = h0 + t / nqt, r0 = first + (t % nqt) * QT;
        qs.load(reinterpret_cast<const T*>(p.q) + (qb + r0) * p.qr + (int64_t)h * p.qh, p.qr, qlen - r0);
        dos.load(reinterpret_cast<const T*>(p.dout) + (qb + r0) * p.dor + (int64_t)h * p.doh, p.dor, qlen - r0);
        if (tid < 2 * QT) {
            const int r = r0 + (tid & (QT - 1));
            const float* src = tid < QT ? p.lse : p.delta;
            st_reg = (tid < QT ? sc.fb : 0.f) - (r < qlen ? src[(int64_t)h * p.Mq + qb + r] : tid < QT ? EMPTY : 0.f);
        }
    };
    auto store = [&](int buf) {
        qs.store(lds[buf][0], tid);
        dos.store(lds[buf][1], tid);
        if (tid < 2 * QT) stat[buf][tid / QT][tid & (QT - 1)] = st_reg;
    };
    if (nt > 0) {
        load(0);
        store(0);
        if (nt > 1) load(1);
    }
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        const int buf = t & 1, r0 = first + (t % nqt) * QT;
        sc.set_head(p, h0 + t / nqt);
        const char *ql = lds[buf][0], *dl = lds[buf][1];
        const int pos0 = off + r0;
        // the wave's keys are all behind the tile's last query: nothing seen
        const bool seen = !p.causal || tile.i0 + w0 < prefix || pos0 + QT - 1 >= tile.i0 + w0;
        if (w0 < tile.n && seen) {
            dkv_block<T, DP, MODE>(dk, dv, ql, dl, stat[buf][0], stat[buf][1], kf, vf, v_l + w0 * ROW, sc, pos0, key, prefix, p.causal && pos0 < tile.i0 + w0 + 31, lane);
        }
        if (t + 1 < nt) {
            store(buf ^ 1);
            if (t + 2 < nt) load(t + 2);
        }
        __syncthreads();
    }
    if (!on) return;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = O::template channel<DP>(d, g, half);
            const float a[4] = {dk[d][4 * g] * back, dk[d][4 * g + 1] * back, dk[d][4 * g + 2] * back, dk[d][4 * g + 3] * back};
            const float b[4] = {dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]};
            if (c >= p.D) continue;
            if (p.parts > 1) {
                PackedVec<float, 4>::store(p.partial + part * p.part_size + at + c, a);
                PackedVec<float, 4>::store(p.partial + (p.parts + part) * p.part_size + at + c, b);
            } else { PackedVec<T, 4>::store(outk + c, a); PackedVec<T, 4>::store(outv + c, b); }
        }
}

// ------------------------------------------------------------------------------------------------ the same for few tiles
// A workgroup takes 32 rows (queries for dQ, keys for dK / dV) and its 4 waves walk the other side in turn, each through its own part of LDS and without
// barriers; their results are added in LDS in the order of the waves.
template <int DP>
__device__ __forceinline__ void put_rows(float* mine, const f32x16 (&y)[DP / 32], float scale, int l31, int half, int (*channel)(int, int, int)) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(mine + l31 * DP + channel(d, g, half)) = f32x4{y[d][4 * g] * scale, y[d][4 * g + 1] * scale, y[d][4 * g + 2] * scale, y[d][4 * g + 3] * scale};
}
template <typename T, int DP, int REGION>
__device__ __forceinline__ void add_rows(T* out, int64_t row_stride, const char (*lds)[REGION], int rows, int D, int tid) {
    const int quads = D / 4;
    for (int u = tid; u < rows * quads; u += 256) {
        const int r = u / quads, c = (u - r * quads) * 4;
        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[w]) + r * DP + c);
            a[0] += x[0]; a[1] += x[1]; a[2] += x[2]; a[3] += x[3];
        }
        PackedVec<T, 4>::store(out + (int64_t)r * row_stride + c, a);
    }
}
template <typename T>
__device__ __forceinline__ void zero_head_rows(T* out, int64_t row_stride, int rows, int D, int tid) {
    for (int u = tid; u < rows * D / 8; u += 256)
        for (int e = 0; e < 8; ++e) out[(int64_t)(u / (D / 8)) * row_stride + u % (D / 8) * 8 + e] = (T)0.f;
}

template <typename T, int DP, int MODE>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void packed_attn_dq_split_kernel(const Args p) {
    typedef Op<T> O;
    constexpr int ROW = DP * (int)sizeof(T) + 16, REGION = 2 * 32 * ROW;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) char lds[4][REGION];
    const int h = blockIdx.x % p.Hq, ti = blockIdx.x / p.Hq / 4, q0 = (blockIdx.x / p.Hq & 3) * 32;
    const PackedTile tile = p.tiles[ti];                         // (beside the count: the list has cap_tiles entries, its rest is not used)
    if (ti >= p.ntiles[1]) return;
    if (q0 >= tile.n) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, half = lane >> 5;
    const int qi = q0 + l31, nq = min(32, tile.n - q0);
    const int64_t row0 = (int64_t)tile.row0 + q0, orow = (int64_t)p.Hq * p.D;
    T* out = reinterpret_cast<T*>(p.dq) + row0 * orow + h * p.D;
    if (tile.doc < 0) { zero_head_rows(out, orow, nq, p.D, tid); return; }
    const int qlen = (int)p.qlen[tile.doc], klen = (int)p.klen[tile.doc];
    const int prefix = p.prefix ? (int)min(max(p.prefix[tile.doc], (int64_t)0), (int64_t)klen) : 0;
    const int64_t kb = p.kbegin[tile.doc];
    const int hk = h / p.G;
    const T* kp = reinterpret_cast<const T*>(p.k) + kb * p.kr + (int64_t)hk * p.kh;
    const T* vp = reinterpret_cast<const T*>(p.v) + kb * p.vr + (int64_t)hk * p.vh;
    char *kl = lds[wave], *vl = lds[wave] + 32 * ROW;
    const int off = klen - qlen + tile.i0;
    const bool on = qi < tile.n;
    const int pos = off + qi, lim = on ? key_limit(pos, klen, prefix, p.causal) : 0;
    const int kmax = max(key_limit(off + q0 + nq - 1, klen, prefix, p.causal), 0), kmin = nq == 32 ? key_limit(off + q0, klen, prefix, p.causal) : 0;
    typename O::Frag qf[O::template NF<DP>], dof[O::template NF<DP>];
    load_frags<T, DP>(dof, row_buffer(reinterpret_cast<const T*>(p.dout) + row0 * p.dor + (int64_t)h * p.doh, p.dor, nq), p.dor, l31, p.D, half);
    float delta = 0.f;
    load_frags<T, DP>(qf, row_buffer(reinterpret_cast<const T*>(p.o) + row0 * orow + h * p.D, orow, nq), orow, l31, p.D, half);
#pragma unroll
    for (int s = 0; s < O::template NF<DP>; ++s)
#pragma unroll
        for (int e = 0; e < O::EPC; ++e) delta = fmaf((float)dof[s][e], (float)qf[s][e], delta);
    if constexpr (!EXACT) {
        load_frags<T, DP>(qf, row_buffer(reinterpret_cast<const T*>(p.rest) + row0 * orow + h * p.D, orow, nq), orow, l31, p.D, half);
#pragma unroll
        for (int s = 0; s < O::template NF<DP>; ++s)
#pragma unroll
            for (int e = 0; e < O::EPC; ++e) delta = fmaf((float)dof[s][e], (float)qf[s][e], delta);
    }
    delta = half_sum(delta);
    if (on && half == 0 && wave == 0) p.delta[(int64_t)h * p.Mq + row0 + l31] = delta;
    load_frags<T, DP>(qf, row_buffer(reinterpret_cast<const T*>(p.q) + row0 * p.qr + (int64_t)h * p.qh, p.qr, nq), p.qr, l31, p.D, half);
    const Score<MODE, EXACT> sc(p, h);
    const float shift = sc.fb - (on ? p.lse[(int64_t)h * p.Mq + row0 + l31] : EMPTY);
    f32x16 acc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = splat(0.f);
    settle(qf);
    settle(dof);
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
        const float dist = (float)(pos - k0 - 4 * half);
        const int left = lim - k0 - 4 * half;
        if (k0 + 32 > kmin) dq_block<T, DP, MODE, true>(acc, kl, vl, qf, dof, sc, delta, shift, dist, left, lane);
        else dq_block<T, DP, MODE, false>(acc, kl, vl, qf, dof, sc, delta, shift, dist, left, lane);
    }
    __builtin_amdgcn_wave_barrier();
    put_rows<DP>(reinterpret_cast<float*>(lds[wave]), acc, p.scale * sc.grad_scale, l31, half, &O::template channel<DP>);
    __syncthreads();
    add_rows<T, DP, REGION>(out, orow, lds, nq, p.D, tid);
}

template <typename T, int DP, int MODE>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DP <= 64 ? 2 : 1) void packed_attn_dkv_split_kernel(const Args p) {
    typedef Op<T> O;
    constexpr bool AHEAD = sizeof(T) == 2 || DP <= 64;                                  // (wide f32 rows requested ahead would not fit the registers)
    constexpr int QT = 32, ROW = DP * (int)sizeof(T) + 16, REGION = 2 * 32 * ROW;
    constexpr bool EXACT = sizeof(T) == 4, VLDS = sizeof(T) == 2;
    __shared__ __attribute__((aligned(16))) char v_l[VLDS ? 32 * ROW : 16];
    __shared__ __attribute__((aligned(16))) char lds[4][REGION];                        // per wave: Q, dO
    __shared__ __attribute__((aligned(16))) float stat[4][2][QT];
    const int hk = blockIdx.x % p.Hk, part = blockIdx.x / p.Hk % p.parts, ti = blockIdx.x / p.Hk / p.parts / 4, k0 = (blockIdx.x / p.Hk / p.parts & 3) * 32;
    const int ndoc = p.ntiles[0];
    if (ti >= p.ntiles[1]) return;
    const PackedTile tile = p.tiles[p.causal && ti < ndoc ? ndoc - 1 - ti : ti];
    if (k0 >= tile.n) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, half = lane >> 5;
    const int nk = min(32, tile.n - k0), i0 = tile.i0 + k0, key = i0 + l31;
    const int64_t row0 = (int64_t)tile.row0 + k0, orow = (int64_t)p.Hk * p.D;
    T* outk = reinterpret_cast<T*>(p.dk) + row0 * orow + hk * p.D;
    T* outv = reinterpret_cast<T*>(p.dv) + row0 * orow + hk * p.D;
    if (tile.doc < 0) {
        if (p.parts == 1) {
            zero_head_rows(outk, orow, nk, p.D, tid);
            zero_head_rows(outv, orow, nk, p.D, tid);
        }
        return;
    }
    float* partial = p.partial + part * p.part_size + row0 * orow + hk * p.D;
    const int qlen = (int)p.qlen[tile.doc], klen = (int)p.klen[tile.doc];
    const int prefix = p.prefix ? (int)min(max(p.prefix[tile.doc], (int64_t)0), (int64_t)klen) : 0;
    const int64_t qb = p.qbegin[tile.doc];
    const int off = klen - qlen;
    const int first = !p.causal || i0 < prefix ? 0 : max(i0 - off, 0);
    typename O::Frag kf[O::template NF<DP>], vf[VLDS ? 1 : O::template NF<DP>];
    load_frags<T, DP>(kf, row_buffer(reinterpret_cast<const T*>(p.k) + row0 * p.kr + (int64_t)hk * p.kh, p.kr, nk), p.kr, l31, p.D, half);
    const T* vrows = reinterpret_cast<const T*>(p.v) + row0 * p.vr + (int64_t)hk * p.vh;
    if constexpr (VLDS) {
        Stage<T, DP, 32, 256> vs(p.vr, p.D, tid);
        vs.load(vrows, p.vr, nk);
        vs.store(v_l, tid);
    } else load_frags<T, DP>(vf, row_buffer(vrows, p.vr, nk), p.vr, l31, p.D, half);
    settle(kf);
    if constexpr (!VLDS) settle(vf);
    __syncthreads();
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) { dk[d] = splat(0.f); dv[d] = splat(0.f); }
    const int nqt = first < qlen ? (qlen - first + QT - 1) / QT : 0, nt = nqt * (p.G / p.parts);
    const int h0 = hk * p.G + part * (p.G / p.parts);                                  // the first of this workgroup's heads
    Score<MODE, EXACT> sc(p, h0);
    Stage<T, DP, QT, 64> qs(p.qr, p.D, lane), dos(p.dor, p.D, lane);
    float st_reg = 0.f;
    char *ql = lds[wave], *dl = lds[wave] + 32 * ROW;
    auto load = [&](int t) {
        const int h = h0 + t / nqt, r0 = first + (t % nqt) * QT;
        qs.load(reinterpret_cast<const T*>(p.q) + (qb + r0) * p.qr + (int64_t)h * p.qh, p.qr, qlen - r0);
        dos.load(reinterpret_cast<const T*>(p.dout) + (qb + r0) * p.dor + (int64_t)h * p.doh, p.dor, qlen - r0);
        const float* src = half == 0 ? p.lse : p.delta;
        st_reg = (half == 0 ? sc.fb : 0.f) - (r0 + l31 < qlen ? src[(int64_t)h * p.Mq + qb + r0 + l31] : half == 0 ? EMPTY : 0.f);
    };
    if (AHEAD && wave < nt) load(wave);
    for (int t = wave; t < nt; t += 4) {
        if (!AHEAD) load(t);
        __builtin_amdgcn_wave_barrier();
        qs.store(ql, lane);
        dos.store(dl, lane);
        stat[wave][half][l31] = st_reg;
        __builtin_amdgcn_wave_barrier();
        if (AHEAD && t + 4 < nt) load(t + 4);
        sc.set_head(p, h0 + t / nqt);
        const int pos0 = off + first + (t % nqt) * QT;
        dkv_block<T, DP, MODE>(dk, dv, ql, dl, stat[wave][0], stat[wave][1], kf, vf, v_l, sc, pos0, key, prefix, p.causal && pos0 < i0 + 31, lane);
    }
    __builtin_amdgcn_wave_barrier();
    put_rows<DP>(reinterpret_cast<float*>(lds[wave]), dk, p.scale * sc.grad_scale, l31, half, &O::template channel<DP>);
    __syncthreads();
    if (p.parts > 1) add_rows<float, DP, REGION>(partial, orow, lds, nk, p.D, tid);
    else add_rows<T, DP, REGION>(outk, orow, lds, nk, p.D, tid);
    __syncthreads();
    put_rows<DP>(reinterpret_cast<float*>(lds[wave]), dv, 1.f, l31, half, &O::template channel<DP>);
    __syncthreads();
    if (p.parts > 1) add_rows<float, DP, REGION>(partial + p.parts * p.part_size, orow, lds, nk, p.D, tid);
    else add_rows<T, DP, REGION>(outv, orow, lds, nk, p.D, tid);
}

// dK and dV from the parts of their heads, in the order of the parts; rows of no document become zeros
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_parts_kernel(const Args p) {
    const PackedTile tile = p.tiles[blockIdx.x];
    if ((int)blockIdx.x >= p.ntiles[1]) return;
    const int64_t row = (int64_t)p.Hk * p.D, first = tile.row0 * row;
    const int quads = (int)(tile.n * row / 4);
    T* out = reinterpret_cast<T*>(blockIdx.y ? p.dv : p.dk);
    const float* in = p.partial + blockIdx.y * p.parts * p.part_size;
    for (int u = blockIdx.z * 256 + threadIdx.x; u < quads; u += 256 * gridDim.z) {
        float a[4] = {0.f, 0.f, 0.f, 0.f};
        if (tile.doc >= 0)
            for (int i = 0; i < p.parts; ++i) {
                const float4 v = *reinterpret_cast<const float4*>(in + i * p.part_size + first + 4 * (int64_t)u);
                a[0] += v.x; a[1] += v.y; a[2] += v.z; a[3] += v.w;
            }
        PackedVec<T, 4>::store(out + first + 4 * (int64_t)u, a);
    }
}

// dK / dV: waves that share 32 keys, and parts the query heads of a key head are cut into, where the workgroups would not fill the chip evenly (one part:
// the sum over the heads stays in registers).  16 heads sharing 4, causal documents of up to 8192 rows, 568 tiles of up to 1024 steps: 2.83 ms in one part,
// 2.46 ms and 0.11 ms for the sums in four.  The waves that share 32 keys are four times as many workgroups already: parts only below one a CU.
struct KeyPlan { bool split; int parts; };
KeyPlan plan_keys(int64_t rows, int64_t docs, int64_t Hk, int64_t G, int64_t qlongest, int64_t D, bool f32) {
    KeyPlan r = {split_waves(rows, docs, Hk, qlongest * G, f32, padded_width(D) > 64), 1};
    const int64_t n = (rows / PACKED_TILE + docs / 2) * Hk * (r.split ? 4 : 1), want = r.split ? 256 : 2048;
    while (r.parts < G && n * r.parts < want) { do ++r.parts; while (G % r.parts); }
    return r;
}

template <typename T, int DP>
void launch(Args p, const PackedTile* ktiles, const int* kntiles, int kcap, hipStream_t s) {
    const int mode = score_mode(p, sizeof(T) == 2);
    Args pk = p;
    pk.tiles = ktiles; pk.ntiles = kntiles; pk.cap_tiles = kcap;
    const bool sq = split_waves(p.Mq, p.docs, p.Hq, p.klongest, sizeof(T) == 4, DP > 64), sk = plan_keys(p.Mk, p.docs, p.Hk, p.G, p.qlongest, p.D, sizeof(T) == 4).split;
    const dim3 gq((unsigned)(p.cap_tiles * p.Hq * (sq ? 4 : 1))), gk((unsigned)(kcap * p.Hk * p.parts * (sk ? 4 : 1)));
#define L(M_)                                                                                       \
    if (sq) hipLaunchKernelGGL((packed_attn_dq_split_kernel<T, DP, M_>), gq, dim3(256), 0, s, p);    \
    else hipLaunchKernelGGL((packed_attn_dq_kernel<T, DP, M_>), gq, dim3(256), 0, s, p);             \
    if (sk) hipLaunchKernelGGL((packed_attn_dkv_split_kernel<T, DP, M_>), gk, dim3(256), 0, s, pk);  \
    else hipLaunchKernelGGL((packed_attn_dkv_kernel<T, DP, M_>), gk, dim3(256), 0, s, pk)
    if constexpr (sizeof(T) == 2) {
        if (mode == (CAP | WIDE)) { L(CAP | WIDE); } else if (mode == (CAP | SLOPE | WIDE)) { L(CAP | SLOPE | WIDE); }
    }
    if (mode == 0) { L(0); } else if (mode == 1) { L(1); } else if (mode == 2) { L(2); } else if (mode == 3) { L(3); }
#undef L
    if (p.parts > 1) hipLaunchKernelGGL((packed_attn_parts_kernel<T>), dim3((unsigned)kcap, 2, 4), dim3(256), 0, s, pk);
}
template <typename T>
void launch_width(const Args& p, const PackedTile* kt, const int* kn, int kcap, hipStream_t s) {
    switch (padded_width(p.D)) {
        case 32: launch<T, 32>(p, kt, kn, kcap, s); break;
        case 64: launch<T, 64>(p, kt, kn, kcap, s); break;
        case 96: launch<T, 96>(p, kt, kn, kcap, s); break;
        default: launch<T, 128>(p, kt, kn, kcap, s);
    }
}
}  // namespace

// Bytes of the workspace of the backward (0: none needed).
extern "C" int64_t osp_packed_attention_bwd_workspace_bytes(int64_t docs, int64_t qlongest, int64_t Mk, int64_t Hq, int64_t Hk, int64_t D, int64_t bf16) {
    if (docs <= 0 || Mk <= 0 || Hk <= 0 || Hq <= 0 || D <= 0) return 0;
    const int64_t parts = plan_keys(Mk, docs, Hk, Hq / Hk, qlongest, D, !bf16).parts;
    return parts > 1 ? 2 * parts * Mk * Hk * D * 4 : 0;
}

extern "C" int osp_packed_attention_bwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v,
                                        int64_t v_row, int64_t v_head, const void* o, const void* rest, const float* lse, const void* dout, int64_t do_row,
                                        int64_t do_head, int64_t bf16, void* dq, void* dk, void* dv, float* delta, void* workspace, const int64_t* qbegin,
                                        const int64_t* qlen, const int32_t* qtiles, const int32_t* qntiles, int64_t qcap, const int64_t* kbegin,
                                        const int64_t* klen, const int32_t* ktiles, const int32_t* kntiles, int64_t kcap, const int64_t* prefix,
                                        const float* slopes, int64_t docs, int64_t qlongest, int64_t klongest, int64_t Mq, int64_t Mk,
                                        int64_t Hq, int64_t Hk, int64_t D, float scale, float softcap, int64_t causal,
                                        hipStream_t stream) {
    OSP_CHECK_ARG(q && k && v && o && (rest || !bf16) && lse && dout && dq && dk && dv && delta && qbegin && qlen && qtiles && qntiles && kbegin && klen && ktiles && kntiles,
                  "null pointer");
    OSP_CHECK_ARG(Hk > 0 && Hq > 0 && Hq % Hk == 0 && Hq <= 65536, "query heads must be a multiple of the key heads");
    OSP_CHECK_ARG(D > 0 && D <= 128 && D % 8 == 0, "head width must be a multiple of 8, at most 128");
    const int E = bf16 ? 8 : 4;
    OSP_CHECK_ARG(q_row % E == 0 && q_head % E == 0 && k_row % E == 0 && k_head % E == 0 && v_row % E == 0 && v_head % E == 0 && do_row % E == 0 &&
                  do_head % E == 0 && packed_aligned(q, 16) && packed_aligned(k, 16) && packed_aligned(v, 16) && packed_aligned(dout, 16) &&
                  packed_aligned(o, 16) && packed_aligned(dq, 16) && packed_aligned(dk, 16) && packed_aligned(dv, 16), "rows and heads must start on 16 bytes");
    OSP_CHECK_ARG(qcap > 0 && kcap > 0 && qcap * Hq < (int64_t)1 << 29 && kcap * Hk < (int64_t)1 << 29 && scale > 0.f && softcap >= 0.f && (causal || !prefix),
                  "bad tile list, cap or mask");
    OSP_CHECK_ARG(row_stride_ok(Hq * D, D, bf16) && row_stride_ok(q_row, D, bf16) && row_stride_ok(k_row, D, bf16) && row_stride_ok(v_row, D, bf16) && row_stride_ok(do_row, D, bf16), "row strides must lie between the head width and 2^24 bytes");
    Args p = {};
    p.q = q; p.k = k; p.v = v; p.o = o; p.rest = const_cast<void*>(rest); p.dout = dout; p.dq = dq; p.dk = dk; p.dv = dv; p.lse = const_cast<float*>(lse); p.delta = delta;
    p.qr = q_row; p.qh = q_head; p.kr = k_row; p.kh = k_head; p.vr = v_row; p.vh = v_head; p.dor = do_row; p.doh = do_head;
    p.qbegin = qbegin; p.qlen = qlen; p.kbegin = kbegin; p.klen = klen; p.tiles = reinterpret_cast<const PackedTile*>(qtiles); p.ntiles = qntiles;
    p.prefix = prefix; p.slopes = slopes; p.Mq = Mq; p.Mk = Mk; p.docs = docs; p.qlongest = qlongest; p.klongest = klongest; p.cap_tiles = (int)qcap; p.Hq = (int)Hq; p.Hk = (int)Hk; p.G = (int)(Hq / Hk); p.D = (int)D;
    p.causal = (int)(causal != 0); p.scale = scale; p.softcap = softcap;
    p.parts = plan_keys(Mk, docs, Hk, Hq / Hk, qlongest, D, !bf16).parts;
    p.part_size = Mk * Hk * D;
    p.partial = reinterpret_cast<float*>(workspace);
    OSP_CHECK_ARG(p.parts == 1 || (workspace && packed_aligned(workspace, 16)), "workspace missing: osp_packed_attention_bwd_workspace_bytes");
    OSP_CHECK_ARG(kcap * Hk * p.parts < (int64_t)1 << 29, "too many tiles");
    const PackedTile* kt = reinterpret_cast<const PackedTile*>(ktiles);
    if (bf16) launch_width<__bf16>(p, kt, kntiles, (int)kcap, stream); else launch_width<float>(p, kt, kntiles, (int)kcap, stream);
    OSP_LAUNCH_CHECK();
    return OSP_OK;
}
