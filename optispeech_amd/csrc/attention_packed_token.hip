// Attention over documents for few queries against many keys (new tokens over a cache), no gradient: the keys are split over workgroups.
// Scores and masks: attention_packed_common.h.
//
// Bound: HBM, the cache is read once.  A workgroup takes one key head and `chunk` keys of one document for all the queries that read them: the
// (queries x heads of the group) are the 32 columns of its score tiles, so shared key heads cost their bytes once.  Each of its 4 waves walks
// its own tiles of 32 keys through its own part of LDS, without barriers: rows are requested into registers one tile ahead (16 KB per wave
// in flight), stored to LDS, and read back as matrix operands.  The waves' results meet in LDS at the end, the splits' (maximum, sum, unscaled
// output) go to a workspace in f32, and a second launch joins them in the order of the splits.
//
// Measured (bf16): 48 requests of 1 .. 16384 keys, 16 heads of 128 sharing 2: 457 MB in 95.5 us (4.8 TB/s; a copy reaches 5.1) and 6 us for the join;  8 streams
// of up to 800 keys, 2 heads: 7.8 + 3.9 us, latency.
#include "attention_packed_common.h"

namespace {
using namespace pattn;

template <typename T, int DP, int MODE>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void packed_attn_token_kernel(const Args p, int chunk, int nsplit, float* __restrict__ po, float* __restrict__ pm) {
    typedef Op<T> O;
    constexpr int ROW = DP * (int)sizeof(T) + 16, REGION = 2 * 32 * ROW;
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ __attribute__((aligned(16))) char lds[4][REGION];                        // per wave: K, V; at the end its output
    __shared__ float ml[4][2][32];
    static_assert(REGION >= 32 * DP * 4, "a wave's output fits its part");
    const int split = blockIdx.x, hk = blockIdx.y, doc = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, half = lane >> 5;
    const int qlen = (int)p.qlen[doc], klen = (int)p.klen[doc];
    const int k_lo = split * chunk, k_hi = split == nsplit - 1 ? klen : min(klen, k_lo + chunk);   // (the last split takes what the host's bound missed)
    if (qlen <= 0 || (split > 0 && k_lo >= klen)) return;
    const int prefix = p.prefix ? (int)min(max(p.prefix[doc], (int64_t)0), (int64_t)klen) : 0;
    const int64_t kb = p.kbegin[doc], qb = p.qbegin[doc];
    const T* kp = reinterpret_cast<const T*>(p.k) + kb * p.kr + (int64_t)hk * p.kh;
    const T* vp = reinterpret_cast<const T*>(p.v) + kb * p.vr + (int64_t)hk * p.vh;
    char *kl = lds[wave], *vl = lds[wave] + 32 * ROW;
    const int cols = qlen * p.G;
    for (int c0 = 0; c0 < cols; c0 += 32) {                                            // more than 32 columns: the keys are walked again
        const int c = c0 + l31, g = c / qlen, i = c - g * qlen;
        const bool on = c < cols;
        const int h = hk * p.G + (on ? g : 0);
        const int64_t qrow = qb + (on ? i : 0);
        typename O::Frag qf[O::template NF<DP>];
        const T* qp = reinterpret_cast<const T*>(p.q) + qrow * p.qr + (int64_t)h * p.qh;     // rows of several heads and queries: no common buffer
#pragma unroll
        for (int s = 0; s < O::template NF<DP>; ++s) {
            const int d = (2 * s + half) * O::EPC;
            typename O::Frag x = {};
            if (on && d < p.D) x = *reinterpret_cast<const typename O::Frag*>(qp + d);
            qf[s] = x;
        }
        const Score<MODE, EXACT> sc(p, h);
        const int pos = klen - qlen + i, lim = on ? key_limit(pos, klen, prefix, p.causal) : 0;
        f32x16 oacc[DP / 32];
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[d][e] = 0.f;
        settle(qf);
        float m_run = NONE, l_run = 0.f;
        Stage<T, DP, 32, 64> ks(p.kr, p.D, lane), vs(p.vr, p.D, lane);
        int k0 = k_lo + wave * 32;
        if (k0 < k_hi) { ks.load(kp + (int64_t)k0 * p.kr, p.kr, k_hi - k0); vs.load(vp + (int64_t)k0 * p.vr, p.vr, k_hi - k0); }
        for (; k0 < k_hi; k0 += 128) {
            __builtin_amdgcn_wave_barrier();
            ks.store(kl, lane);
            vs.store(vl, lane);
            __builtin_amdgcn_wave_barrier();
            if (k0 + 128 < k_hi) { ks.load(kp + (int64_t)(k0 + 128) * p.kr, p.kr, k_hi - k0 - 128); vs.load(vp + (int64_t)(k0 + 128) * p.vr, p.vr, k_hi - k0 - 128); }
            f32x16 st = O::template score<DP>(kl, qf, l31, half, splat(0.f));
            const float dist = (float)(pos - k0 - 4 * half);
            const int left = min(lim, k_hi) - k0 - 4 * half;
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int r = (e >> 2) * 8 + (e & 3);
                const float s = sc.penalise(sc.cap(st[e]), dist - (float)r);
                st[e] = r < left ? s : -INFINITY;
                mx = fmaxf(mx, st[e]);
            }
            mx = fmaf(half_max(mx), sc.fa, sc.fb);
            if (__any(mx > m_run + 8.f)) {
                const float m_new = fmaxf(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < DP / 32; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) oacc[d][e] *= alpha;
            }
            typename O::Cols pc;
            const float shift = sc.fb - m_run;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = __builtin_amdgcn_exp2f(fmaf(st[e], sc.fa, shift));
                l_run += x;
                O::set(pc, e, x);
            }
            O::template value<DP>(oacc, pc, vl, lane);
        }
        l_run = half_sum(l_run);
        if (half == 0) { ml[wave][0][l31] = m_run; ml[wave][1][l31] = l_run; }
        __syncthreads();
        float mall = NONE;
#pragma unroll
        for (int w = 0; w < 4; ++w) mall = fmaxf(mall, ml[w][0][l31]);
        const float f = __builtin_amdgcn_exp2f(m_run - mall);
        float* mine = reinterpret_cast<float*>(lds[wave]);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<f32x4*>(mine + l31 * DP + O::template channel<DP>(d, q4, half)) =
                    f32x4{oacc[d][4 * q4] * f, oacc[d][4 * q4 + 1] * f, oacc[d][4 * q4 + 2] * f, oacc[d][4 * q4 + 3] * f};
        __syncthreads();
        const int nc = min(32, cols - c0);
        for (int u = tid; u < nc * DP; u += 256) {
            const int cc = u / DP, d = u - cc * DP;
            const int gg = (c0 + cc) / qlen, ii = c0 + cc - gg * qlen;
            const int64_t slot = ((int64_t)split * p.Mq + qb + ii) * p.Hq + hk * p.G + gg;
            if (d < p.D) {
                float a = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) a += reinterpret_cast<const float*>(lds[w])[u];
                po[slot * p.D + d] = a;
            }
            if (d == 0) {
                float m = NONE, l = 0.f;
                for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w][0][cc]);
                for (int w = 0; w < 4; ++w) l = fmaf(ml[w][1][cc], __builtin_amdgcn_exp2f(ml[w][0][cc] - m), l);
                *reinterpret_cast<float2*>(pm + slot * 2) = make_float2(m, l);
            }
        }
        __syncthreads();
    }
}

// joins the splits of every query row and head; rows of no document become zeros.  D / 4 threads hold a row, groups of them take the splits in turn (their
// loads are in flight together) and meet in LDS, in the order of the groups.
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_join_kernel(const Args p, int chunk, int nsplit, const float* __restrict__ po, const float* __restrict__ pm) {
    __shared__ float4 red_a[256];
    __shared__ float2 red_m[256];
    const PackedTile tile = p.tiles[blockIdx.x];
    if ((int)blockIdx.x >= p.ntiles[1]) return;
    const int h = blockIdx.y, quads = p.D / 4, groups = 256 / quads, g = threadIdx.x / quads, d = (threadIdx.x - g * quads) * 4;
    int n = 0;
    if (tile.doc >= 0) {
        const int klen = (int)p.klen[tile.doc];
        n = max(1, min(nsplit, (klen + chunk - 1) / chunk));
    }
    const int64_t step = p.Mq * p.Hq;
    for (int r = 0; r < tile.n; ++r) {
        const int64_t slot0 = ((int64_t)tile.row0 + r) * p.Hq + h;
        float m = NONE, l = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        if (g < groups) {
#pragma unroll 4
            for (int s = g; s < n; s += groups) {
                const float2 x = *reinterpret_cast<const float2*>(pm + (slot0 + s * step) * 2);
                const float4 y = *reinterpret_cast<const float4*>(po + (slot0 + s * step) * p.D + d);
                const float mn = fmaxf(m, x.x), fo = __builtin_amdgcn_exp2f(m - mn), fn = __builtin_amdgcn_exp2f(x.x - mn);
                m = mn;
                l = l * fo + x.y * fn;
                a = make_float4(a.x * fo + y.x * fn, a.y * fo + y.y * fn, a.z * fo + y.z * fn, a.w * fo + y.w * fn);
            }
        }
        red_a[threadIdx.x] = a;
        red_m[threadIdx.x] = make_float2(m, l);
        __syncthreads();
        if (g == 0) {
            const int live = min(groups, max(n, 1));
            for (int i = 1; i < live; ++i) m = fmaxf(m, red_m[i * quads + threadIdx.x].x);
            l = 0.f;
            a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < live; ++i) {
                const float2 x = red_m[i * quads + threadIdx.x];
                const float4 y = red_a[i * quads + threadIdx.x];
                const float f = __builtin_amdgcn_exp2f(x.x - m);
                l = fmaf(x.y, f, l);
                a = make_float4(fmaf(y.x, f, a.x), fmaf(y.y, f, a.y), fmaf(y.z, f, a.z), fmaf(y.w, f, a.w));
            }
            const float inv = l > 0.f ? 1.f / l : 0.f;
            const float o[4] = {a.x * inv, a.y * inv, a.z * inv, a.w * inv};
            PackedVec<T, 4>::store(reinterpret_cast<T*>(p.out) + slot0 * p.D + d, o);
        }
        __syncthreads();
    }
}

template <typename T, int DP>
void launch(const Args& p, int B, int chunk, int nsplit, float* po, float* pm, hipStream_t s) {
    const dim3 grid((unsigned)nsplit, (unsigned)p.Hk, (unsigned)B);
    const int mode = score_mode(p, sizeof(T) == 2);
#define L(M_) hipLaunchKernelGGL((packed_attn_token_kernel<T, DP, M_>), grid, dim3(256), 0, s, p, chunk, nsplit, po, pm)
    if constexpr (sizeof(T) == 2) {
        if (mode == (CAP | WIDE)) { L(CAP | WIDE); } else if (mode == (CAP | SLOPE | WIDE)) { L(CAP | SLOPE | WIDE); }
    }
    if (mode == 0) { L(0); } else if (mode == 1) { L(1); } else if (mode == 2) { L(2); } else if (mode == 3) { L(3); }
#undef L
    hipLaunchKernelGGL((packed_attn_join_kernel<T>), dim3((unsigned)p.cap_tiles, (unsigned)p.Hq), dim3(256), 0, s, p, chunk, nsplit, po, pm);
}
template <typename T>
void launch_width(const Args& p, int B, int chunk, int nsplit, float* po, float* pm, hipStream_t s) {
    switch (padded_width(p.D)) {
        case 32: launch<T, 32>(p, B, chunk, nsplit, po, pm, s); break;
        case 64: launch<T, 64>(p, B, chunk, nsplit, po, pm, s); break;
        case 96: launch<T, 96>(p, B, chunk, nsplit, po, pm, s); break;
        default: launch<T, 128>(p, B, chunk, nsplit, po, pm, s);
    }
}

// Keys a workgroup takes: enough workgroups to fill the chip several times over, 128 keys (one tile for each of its waves) at least.
int64_t chunk_keys(int64_t B, int64_t Hk, int64_t longest) {
    const int64_t want = 2048;
    int64_t c = cdiv(cdiv(B * Hk * longest, want), 128) * 128;
    return c < 128 ? 128 : c;
}
}  // namespace

// Bytes of the workspace: one f32 output row and two statistics per split, query row and head.
extern "C" int64_t osp_packed_attention_token_workspace_bytes(int64_t B, int64_t Mq, int64_t longest, int64_t Hq, int64_t Hk, int64_t D) {
    if (B <= 0 || Mq <= 0 || longest <= 0 || Hq <= 0 || Hk <= 0 || D <= 0) return 0;
    return cdiv(longest, chunk_keys(B, Hk, longest)) * Mq * Hq * (D + 2) * 4;
}

extern "C" int osp_packed_attention_token(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v,
                                          int64_t v_row, int64_t v_head, int64_t bf16, void* o, void* workspace, const int64_t* qbegin,
                                          const int64_t* qlen, const int32_t* qtiles, const int32_t* qntiles, int64_t qcap, const int64_t* kbegin,
                                          const int64_t* klen, int64_t longest, const int64_t* prefix, const float* slopes, int64_t B, int64_t Mq,
                                          int64_t Hq, int64_t Hk, int64_t D, float scale, float softcap, int64_t causal, hipStream_t stream) {
    OSP_CHECK_ARG(q && k && v && o && workspace && qbegin && qlen && qtiles && qntiles && kbegin && klen, "null pointer");
    OSP_CHECK_ARG(B > 0 && B < 65536 && Mq > 0 && longest > 0 && longest < (int64_t)1 << 31, "1 .. 65535 documents with at least one key in the bound");
    OSP_CHECK_ARG(Hk > 0 && Hq > 0 && Hq % Hk == 0 && Hq < 65536, "query heads must be a multiple of the key heads");
    OSP_CHECK_ARG(D > 0 && D <= 128 && D % 8 == 0, "head width must be a multiple of 8, at most 128");
    const int E = bf16 ? 8 : 4;
    OSP_CHECK_ARG(q_row % E == 0 && q_head % E == 0 && k_row % E == 0 && k_head % E == 0 && v_row % E == 0 && v_head % E == 0 && packed_aligned(q, 16) &&
                  packed_aligned(k, 16) && packed_aligned(v, 16) && packed_aligned(o, 16) && packed_aligned(workspace, 16), "rows and heads must start on 16 bytes");
    OSP_CHECK_ARG(qcap > 0 && qcap < (int64_t)1 << 31 && scale > 0.f && softcap >= 0.f && (causal || !prefix), "bad tile list, cap or mask");
    OSP_CHECK_ARG(row_stride_ok(q_row, D, bf16) && row_stride_ok(k_row, D, bf16) && row_stride_ok(v_row, D, bf16), "row strides must lie between the head width and 2^24 bytes");
    Args p = {};
    p.q = q; p.k = k; p.v = v; p.out = o;
    p.qr = q_row; p.qh = q_head; p.kr = k_row; p.kh = k_head; p.vr = v_row; p.vh = v_head;
    p.qbegin = qbegin; p.qlen = qlen; p.kbegin = kbegin; p.klen = klen; p.tiles = reinterpret_cast<const PackedTile*>(qtiles); p.ntiles = qntiles;
    p.prefix = prefix; p.slopes = slopes; p.Mq = Mq; p.cap_tiles = (int)qcap; p.Hq = (int)Hq; p.Hk = (int)Hk; p.G = (int)(Hq / Hk); p.D = (int)D;
    p.causal = (int)(causal != 0); p.scale = scale; p.softcap = softcap;
    const int64_t chunk = chunk_keys(B, Hk, longest), nsplit = cdiv(longest, chunk);
    float* po = reinterpret_cast<float*>(workspace);
    float* pm = po + nsplit * Mq * Hq * D;
    if (bf16) launch_width<__bf16>(p, (int)B, (int)chunk, (int)nsplit, po, pm, stream);
    else launch_width<float>(p, (int)B, (int)chunk, (int)nsplit, po, pm, stream);
    OSP_LAUNCH_CHECK();
    return OSP_OK;
}
