// Group norm with an activation on packed rows, channels last: y = act(w (x - mean) rstd + b), statistics over a document's rows and a
// group's channels, forward and backward.
//   forward : mean, rstd per (document, group) from sum x and sum x^2
//   backward: z = w xhat + b, dz = dy act'(z), gw = dz w;   dx = rstd (gw - mean(gw) - xhat mean(gw xhat)),
//             dw += sum dz xhat,  db += sum dz   over all documents
// Rows of no document get zeros (y and dx) and add nothing.
//
// Sums: x and x^2 are summed in 64 bits (x^2 of an f32 is exact there; the vector units do 64-bit FMAs at the 32-bit rate and the kernel is bound by HBM),
// and for f32 tensors the mean is kept as two floats, m + rest: rounded to one it would shift every xhat of a group by up to 2^-24 |mean| / deviation.  A
// mean far above the deviation then costs what the 64-bit sums lose, about 2^-53 (mean / deviation)^2 of rstd per addition in a chain (1e-6 where
// the mean is 10^5 deviations), instead of 6e-3.  The backward's per-channel sums run in 32 bits over the rows of one
// workgroup (at most PACKED_TILE) and in 64 bits from there on.  Every sum has one fixed order: no atomics.
//
// Bound: HBM.  Where a document's rows x one slab of groups fit the registers of a workgroup, one launch reads x (and dy) once: see "documents that fit".
// Longer documents and groups that are no whole vectors are read twice, the second time mostly out of the 256 MB last-level cache.  Forward: partial sums per (tile part, group) -> apply, whose workgroups add the few partials of their document
// themselves (a launch of its own does it where a document has many).  Backward: per-channel partials -> per-document sums -> apply, the
// sum of the documents' dw / db riding on the last launch.
//
// Measured: 37 k rows x 384 channels bf16, 8 groups, silu: forward 18.3 us (3.1 TB/s), backward 35.2 + 3.9 us (the silu and its slope, evaluated twice, take 11 of
// them);  23 k rows x 256 channels f32, 32 groups, gelu: 17.4 and 30.9 + 4.0 us.  Twice through memory instead: 28 and 43 us, 25 and 45 us.
#include "packed_common.h"

namespace {

constexpr int NTH = 256, MAXC = 2048;

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

// EXACT: f32 tensors take the library's expf / erff; bf16 results take one v_exp_f32 / v_rcp_f32 and the polynomial erf (<= 1.5e-7)
template <int ACT, bool EXACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == ACT_RELU) return fmaxf(z, 0.f);
    if constexpr (ACT == ACT_GELU) return EXACT ? gelu_f(z) : gelu_fast_f(z);
    if constexpr (ACT == ACT_SILU) {
        if constexpr (EXACT) return z / (1.f + expf(-z));
        return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
    }
    return z;
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if constexpr (ACT == ACT_GELU) {
        if constexpr (EXACT) {
            const float cdf = 0.5f * (1.0f + erff(z * 0.70710678118654752440f));
            return fmaf(z * 0.39894228040143267794f, expf(-0.5f * z * z), cdf);
        }
        return gelu_grad_fast_f(z);
    }
    if constexpr (ACT == ACT_SILU) {
        float s;
        if constexpr (EXACT) s = 1.f / (1.f + expf(-z)); else s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
        return s * fmaf(z, 1.f - s, 1.f);
    }
    return 1.f;
}

struct NormArgs {
    const void* x; int64_t ldx;
    const void* dy; int64_t lddy;
    const float *w, *b;
    void* out;                                  // y or dx, (M, C) contiguous
    float *mean, *rstd, *rest;                  // (B, G); rest: the mean's part below f32, for f32 tensors
    double* part;                               // forward: (slots, G, 2)
    float* cpart;                               // backward: (slots, C, 2)
    double* dsum;                               // backward: (B, C, 2) sums of dz, dz xhat
    float* coef;                                // backward: (B, G, 2) mean(gw), mean(gw xhat)
    float *dw, *db;                             // added to where add_w / add_b, written otherwise
    int add_w, add_b;
    const int64_t *begin, *len;
    const int* base;
    const PackedTile* tiles;
    const int* ntiles;
    int B, C, G, cap, sub;                      // sub: parts a tile is cut into (rows PACKED_TILE / sub)
    float eps;
};

// threads -> (row lane, channel vector): nx threads along the channels, ny rows at a time
struct Lanes { int nx, ny, cx, ry; };
__device__ __forceinline__ Lanes lanes_of(int nvec) {
    Lanes l;
    l.nx = min(nvec, NTH);
    l.ny = NTH / l.nx;
    l.ry = threadIdx.x / l.nx;
    l.cx = threadIdx.x - l.ry * l.nx;
    return l;
}

// n elements from y on become zeros, 16 bytes at a time where they start on 16 bytes
template <typename T>
__device__ __forceinline__ void zero_rows(T* y, int64_t n) {
    constexpr int E = 16 / (int)sizeof(T);
    const int64_t m = reinterpret_cast<uintptr_t>(y) % 16 == 0 ? n / E : 0;
    for (int64_t i = threadIdx.x; i < m; i += blockDim.x) reinterpret_cast<float4*>(y)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int64_t i = m * E + threadIdx.x; i < n; i += blockDim.x) y[i] = (T)0.f;
}

// sum over the lanes of aligned groups of L (a power of two)
__device__ __forceinline__ double lane_group_sum(double v, int L) {
    for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// x - mean: f32 tensors take the mean's second part off too (bf16 values resolve 2^-9 of the mean: its rounding to f32 is far below)
template <typename T>
__device__ __forceinline__ float centre(float x, float m, float rest) {
    if constexpr (sizeof(T) == 4) return (x - m) - rest;
    return x - m;
}

// a document's statistics from its partials; results for every group in LDS: G means, G rstd, G rests
__device__ __forceinline__ void doc_stats(const NormArgs& p, int doc, int64_t rows, float* stat_l) {
    const int nslots = (int)((rows + PACKED_TILE - 1) / PACKED_TILE) * p.sub;
    const double* part = p.part + (int64_t)p.base[doc] * p.sub * p.G * 2;
    int L = 1;
    while (L < 64 && 2 * L * p.G <= NTH) L <<= 1;
    const double count = (double)rows * (double)(p.C / p.G);
    for (int g0 = 0; g0 < p.G; g0 += NTH / L) {
        const int g = g0 + (int)threadIdx.x / L, l = threadIdx.x % L;
        double s = 0.0, q = 0.0;
        if (g < p.G)
            for (int i = l; i < nslots; i += L) {
                const double2 v = *reinterpret_cast<const double2*>(part + ((int64_t)i * p.G + g) * 2);
                s += v.x; q += v.y;
            }
        s = lane_group_sum(s, L);
        q = lane_group_sum(q, L);
        if (g < p.G && l == 0) {
            const double m = s / count, var = fmax(q / count - m * m, 0.0);
            stat_l[g] = (float)m;
            stat_l[p.G + g] = (float)(1.0 / sqrt(var + (double)p.eps));
            stat_l[2 * p.G + g] = (float)(m - (double)(float)m);
        }
    }
    __syncthreads();
}

// ------------------------------------------------------------------------------------------------ forward: partial sums
template <typename T, int V>
__global__ __launch_bounds__(NTH) void gn_stats_kernel(const NormArgs p) {
    extern __shared__ double2 smem[];           // [ny][chunk] then [C]
    if ((int)blockIdx.x >= p.ntiles[0]) return;
    const PackedTile tile = p.tiles[blockIdx.x];
    const int step = PACKED_TILE / p.sub, lo = blockIdx.y * step, hi = min(tile.n, lo + step);
    const Lanes l = lanes_of(p.C / V);
    double2* chan = smem + NTH * V;
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)tile.row0 * p.ldx;
    for (int c0 = 0; c0 < p.C / V; c0 += l.nx) {
        const int cv = c0 + l.cx;
        double s[V], q[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { s[i] = 0.0; q[i] = 0.0; }
        const bool on = l.ry < l.ny && cv < p.C / V;
        if (on) {
#pragma unroll 4
            for (int r = lo + l.ry; r < hi; r += l.ny) {
                float f[V];
                PackedVec<T, V>::load(f, x + (int64_t)r * p.ldx + cv * V);
#pragma unroll
                for (int i = 0; i < V; ++i) { const double d = (double)f[i]; s[i] += d; q[i] = fma(d, d, q[i]); }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) smem[(l.ry * l.nx + l.cx) * V + i] = make_double2(s[i], q[i]);
        }
        __syncthreads();
        const int chunk = min(l.nx, p.C / V - c0) * V;
        for (int c = threadIdx.x; c < chunk; c += NTH) {
            double2 a = smem[c];
            for (int r = 1; r < l.ny; ++r) { const double2 v = smem[r * l.nx * V + c]; a.x += v.x; a.y += v.y; }
            chan[c0 * V + c] = a;
        }
        __syncthreads();
    }
    const int cg = p.C / p.G;
    int L = 1;
    while (L < 64 && 2 * L * p.G <= NTH) L <<= 1;
    double* part = p.part + ((int64_t)(p.base[tile.doc] + tile.i0 / PACKED_TILE) * p.sub + blockIdx.y) * p.G * 2;
    for (int g0 = 0; g0 < p.G; g0 += NTH / L) {
        const int g = g0 + (int)threadIdx.x / L, ln = threadIdx.x % L;
        double s = 0.0, q = 0.0;
        if (g < p.G)
            for (int i = ln; i < cg; i += L) { const double2 v = chan[g * cg + i]; s += v.x; q += v.y; }
        s = lane_group_sum(s, L);
        q = lane_group_sum(q, L);
        if (g < p.G && ln == 0) *reinterpret_cast<double2*>(part + g * 2) = make_double2(s, q);
    }
}

// statistics of one document per workgroup (where a document has too many partials for every apply workgroup to add them)
__global__ __launch_bounds__(NTH) void gn_finish_kernel(const NormArgs p) {
    __shared__ float stat_l[3 * MAXC];
    const int doc = blockIdx.x;
    const int64_t rows = p.len[doc];
    if (rows <= 0) {
        for (int g = threadIdx.x; g < p.G; g += NTH) { p.mean[(int64_t)doc * p.G + g] = 0.f; p.rstd[(int64_t)doc * p.G + g] = 0.f; p.rest[(int64_t)doc * p.G + g] = 0.f; }
        return;
    }
    doc_stats(p, doc, rows, stat_l);
    for (int g = threadIdx.x; g < p.G; g += NTH) {
        p.mean[(int64_t)doc * p.G + g] = stat_l[g];
        p.rstd[(int64_t)doc * p.G + g] = stat_l[p.G + g];
        p.rest[(int64_t)doc * p.G + g] = stat_l[2 * p.G + g];
    }
}


// ------------------------------------------------------------------------------------------------ forward: apply
template <typename T, int V, int ACT, bool DIRECT>
__global__ __launch_bounds__(NTH) void gn_apply_kernel(const NormArgs p) {
    extern __shared__ float stat[];             // [G] mean, [G] rstd, [G] rest
    if ((int)blockIdx.x >= p.ntiles[1]) return;
    const PackedTile tile = p.tiles[blockIdx.x];
    const int step = PACKED_TILE / p.sub, lo = blockIdx.y * step, hi = min(tile.n, lo + step);
    if (lo >= hi) return;
    T* y = reinterpret_cast<T*>(p.out) + (int64_t)tile.row0 * p.C;
    if (tile.doc < 0) { zero_rows(y + (int64_t)lo * p.C, (int64_t)(hi - lo) * p.C); return; }
    if (DIRECT) {
        doc_stats(p, tile.doc, p.len[tile.doc], stat);
        if (tile.i0 == 0 && lo == 0)
            for (int g = threadIdx.x; g < p.G; g += NTH) {
                p.mean[(int64_t)tile.doc * p.G + g] = stat[g];
                p.rstd[(int64_t)tile.doc * p.G + g] = stat[p.G + g];
                p.rest[(int64_t)tile.doc * p.G + g] = stat[2 * p.G + g];
            }
    }
    const float* mean = DIRECT ? stat : p.mean + (int64_t)tile.doc * p.G;
    const float* rstd = DIRECT ? stat + p.G : p.rstd + (int64_t)tile.doc * p.G;
    const float* rest = DIRECT ? stat + 2 * p.G : p.rest + (int64_t)tile.doc * p.G;
    const Lanes l = lanes_of(p.C / V);
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)tile.row0 * p.ldx;
    const int cg = p.C / p.G;
    for (int cv = l.cx; cv < p.C / V && l.ry < l.ny; cv += l.nx) {
        float m[V], rs[V], ml[V], w[V], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = cv * V + i, g = c / cg;
            m[i] = mean[g]; rs[i] = rstd[g]; ml[i] = rest[g]; w[i] = p.w[c]; b[i] = p.b[c];
        }
#pragma unroll 4
        for (int r = lo + l.ry; r < hi; r += l.ny) {
            float f[V];
            PackedVec<T, V>::load(f, x + (int64_t)r * p.ldx + cv * V);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = act_value<ACT, sizeof(T) == 4>(fmaf(centre<T>(f[i], m[i], ml[i]) * rs[i], w[i], b[i]));
            PackedVec<T, V>::store(y + (int64_t)r * p.C + cv * V, f);
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward: per-channel partial sums
template <typename T, int V, int ACT>
__global__ __launch_bounds__(NTH) void gn_bwd_sums_kernel(const NormArgs p) {
    __shared__ float2 stage[NTH * V];
    if ((int)blockIdx.x >= p.ntiles[0]) return;
    const PackedTile tile = p.tiles[blockIdx.x];
    const int step = PACKED_TILE / p.sub, lo = blockIdx.y * step, hi = min(tile.n, lo + step);
    const Lanes l = lanes_of(p.C / V);
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)tile.row0 * p.ldx;
    const T* dy = reinterpret_cast<const T*>(p.dy) + (int64_t)tile.row0 * p.lddy;
    const float *mean = p.mean + (int64_t)tile.doc * p.G, *rstd = p.rstd + (int64_t)tile.doc * p.G, *rest = p.rest + (int64_t)tile.doc * p.G;
    float2* out = reinterpret_cast<float2*>(p.cpart) + ((int64_t)(p.base[tile.doc] + tile.i0 / PACKED_TILE) * p.sub + blockIdx.y) * p.C;
    const int cg = p.C / p.G;
    for (int c0 = 0; c0 < p.C / V; c0 += l.nx) {
        const int cv = c0 + l.cx;
        if (l.ry < l.ny && cv < p.C / V) {
            float m[V], rs[V], ml[V], w[V], b[V], s[V], q[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = cv * V + i, g = c / cg;
                m[i] = mean[g]; rs[i] = rstd[g]; ml[i] = rest[g]; w[i] = p.w[c]; b[i] = p.b[c]; s[i] = 0.f; q[i] = 0.f;
            }
#pragma unroll 2
            for (int r = lo + l.ry; r < hi; r += l.ny) {
                float f[V], d[V];
                PackedVec<T, V>::load(f, x + (int64_t)r * p.ldx + cv * V);
                PackedVec<T, V>::load(d, dy + (int64_t)r * p.lddy + cv * V);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float hat = centre<T>(f[i], m[i], ml[i]) * rs[i];
                    const float dz = d[i] * act_slope<ACT, sizeof(T) == 4>(fmaf(hat, w[i], b[i]));
                    s[i] += dz;
                    q[i] = fmaf(dz, hat, q[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) stage[(l.ry * l.nx + l.cx) * V + i] = make_float2(s[i], q[i]);
        }
        __syncthreads();
        const int chunk = min(l.nx, p.C / V - c0) * V;
        for (int c = threadIdx.x; c < chunk; c += NTH) {
            float2 a = stage[c];
            for (int r = 1; r < l.ny; ++r) { const float2 v = stage[r * l.nx * V + c]; a.x += v.x; a.y += v.y; }
            out[c0 * V + c] = a;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ backward: a document's sums
// grid (documents, group chunks): a chunk is as many whole groups as fit 64 channels (one group where it is wider); 64 channels x 8 slot lanes
__global__ __launch_bounds__(512) void gn_bwd_docs_kernel(const NormArgs p, int gchunk) {
    extern __shared__ double2 chan[];           // [gchunk * C / G]
    __shared__ double2 red[8][64];
    const int doc = blockIdx.x, cg = p.C / p.G, g0 = blockIdx.y * gchunk, ng = min(gchunk, p.G - g0);
    const int64_t rows = p.len[doc];
    const int nslots = (int)((rows + PACKED_TILE - 1) / PACKED_TILE) * p.sub;
    const float2* part = reinterpret_cast<const float2*>(p.cpart) + (int64_t)p.base[doc] * p.sub * p.C;
    const int lane = threadIdx.x & 63, sl = threadIdx.x >> 6;
    double2* out = reinterpret_cast<double2*>(p.dsum) + (int64_t)doc * p.C;
    for (int c0 = 0; c0 < ng * cg; c0 += 64) {
        const int c = c0 + lane;
        double a = 0.0, b = 0.0;
        if (c < ng * cg) {
#pragma unroll 4
            for (int i = sl; i < nslots; i += 8) { const float2 v = part[(int64_t)i * p.C + g0 * cg + c]; a += v.x; b += v.y; }
        }
        red[sl][lane] = make_double2(a, b);
        __syncthreads();
        if (sl == 0 && c < ng * cg) {
            for (int i = 1; i < 8; ++i) { a += red[i][lane].x; b += red[i][lane].y; }
            out[g0 * cg + c] = make_double2(a, b);
            const double w = (double)p.w[g0 * cg + c];
            chan[c] = make_double2(w * a, w * b);
        }
        __syncthreads();
    }
    const double inv = rows > 0 ? 1.0 / ((double)rows * (double)cg) : 0.0;
    for (int g = threadIdx.x >> 6; g < ng; g += 8) {
        double a = 0.0, b = 0.0;
        for (int i = lane; i < cg; i += 64) { a += chan[g * cg + i].x; b += chan[g * cg + i].y; }
        a = lane_group_sum(a, 64);
        b = lane_group_sum(b, 64);
        if (lane == 0) {
            float* o = p.coef + ((int64_t)doc * p.G + g0 + g) * 2;
            o[0] = (float)(a * inv);
            o[1] = (float)(b * inv);
        }
    }
}

__device__ __forceinline__ void weight_sums(const NormArgs& p, int c0) {
    __shared__ double2 red[4][64];
    const int lane = threadIdx.x & 63, sl = threadIdx.x >> 6, c = c0 + lane;
    double a = 0.0, b = 0.0;
    if (c < p.C) {
#pragma unroll 4
        for (int d = sl; d < p.B; d += 4) { const double2 v = reinterpret_cast<const double2*>(p.dsum)[(int64_t)d * p.C + c]; a += v.x; b += v.y; }
    }
    red[sl][lane] = make_double2(a, b);
    __syncthreads();
    if (sl == 0 && c < p.C) {
        for (int i = 1; i < 4; ++i) { a += red[i][lane].x; b += red[i][lane].y; }
        if (p.db) p.db[c] = (float)a + (p.add_b ? p.db[c] : 0.f);
        if (p.dw) p.dw[c] = (float)b + (p.add_w ? p.dw[c] : 0.f);
    }
}

// ------------------------------------------------------------------------------------------------ backward: dx, and dw / db behind the tiles
template <typename T, int V, int ACT>
__global__ __launch_bounds__(NTH) void gn_bwd_apply_kernel(const NormArgs p) {
    if ((int)blockIdx.x >= p.cap) {              // the last workgroups
        if (!blockIdx.y) weight_sums(p, ((int)blockIdx.x - p.cap) * 64);
        return;
    }
    if ((int)blockIdx.x >= p.ntiles[1] || !p.out) return;
    const PackedTile tile = p.tiles[blockIdx.x];
    const int step = PACKED_TILE / p.sub, lo = blockIdx.y * step, hi = min(tile.n, lo + step);
    if (lo >= hi) return;
    T* dx = reinterpret_cast<T*>(p.out) + (int64_t)tile.row0 * p.C;
    if (tile.doc < 0) { zero_rows(dx + (int64_t)lo * p.C, (int64_t)(hi - lo) * p.C); return; }
    const Lanes l = lanes_of(p.C / V);
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)tile.row0 * p.ldx;
    const T* dy = reinterpret_cast<const T*>(p.dy) + (int64_t)tile.row0 * p.lddy;
    const float *mean = p.mean + (int64_t)tile.doc * p.G, *rstd = p.rstd + (int64_t)tile.doc * p.G, *rest = p.rest + (int64_t)tile.doc * p.G;
    const float2* coef = reinterpret_cast<const float2*>(p.coef) + (int64_t)tile.doc * p.G;
    const int cg = p.C / p.G;
    for (int cv = l.cx; cv < p.C / V && l.ry < l.ny; cv += l.nx) {
        float m[V], rs[V], ml[V], w[V], b[V], c1[V], c2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = cv * V + i, g = c / cg;
            m[i] = mean[g]; rs[i] = rstd[g]; ml[i] = rest[g]; w[i] = p.w[c]; b[i] = p.b[c];
            const float2 k = coef[g];
            c1[i] = k.x; c2[i] = k.y;
        }
#pragma unroll 2
        for (int r = lo + l.ry; r < hi; r += l.ny) {
            float f[V], d[V];
            PackedVec<T, V>::load(f, x + (int64_t)r * p.ldx + cv * V);
            PackedVec<T, V>::load(d, dy + (int64_t)r * p.lddy + cv * V);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float hat = centre<T>(f[i], m[i], ml[i]) * rs[i];
                const float gw = d[i] * act_slope<ACT, sizeof(T) == 4>(fmaf(hat, w[i], b[i])) * w[i];
                f[i] = rs[i] * (gw - c1[i] - hat * c2[i]);
            }
            PackedVec<T, V>::store(dx + (int64_t)r * p.C + cv * V, f);
        }
    }
}

// ------------------------------------------------------------------------------------------------ documents that fit a workgroup's registers
// One workgroup = one document x one slab of whole groups (64 bytes of a row or more where a few groups give that).  Its RT threads (512, two workgroups to
// a CU; 1024 where 512 would keep more than 7 vectors each) load the slab into registers once (NR vectors of 16 bytes, all in flight together), reduce, and write the result: x is read once and nothing passes
// through memory.  Slabs of one document are given to one XCD, whose L2 then serves the parts of a line that neighbouring slabs read.
// Rows beyond NR * ny (a bound `longest` that is too small) are read from memory in both passes.
constexpr int GAP_WGS = 64;

struct Slab { int nslab, gs, sc; };              // slabs of a row, groups and channels of one

__device__ __forceinline__ bool slab_of(const NormArgs& p, const Slab& sl, int& doc, int& c0) {
    const int n = p.B * sl.nslab, per = (n + 7) / 8;                       // XCD = workgroup % 8: eight contiguous runs of (document, slab)
    const int at = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per || at >= n) return false;
    doc = at / sl.nslab;
    c0 = (at - doc * sl.nslab) * sl.sc;
    return true;
}
template <typename T>
__device__ __forceinline__ void zero_gaps(const NormArgs& p, int first) {  // the workgroups behind the slabs: rows of no document
    for (int t = p.ntiles[0] + (int)blockIdx.x - first; t < p.ntiles[1]; t += GAP_WGS) {
        const PackedTile tile = p.tiles[t];
        zero_rows(reinterpret_cast<T*>(p.out) + (int64_t)tile.row0 * p.C, (int64_t)tile.n * p.C);
    }
}

// sums of (a, b) over the threads of each group of the slab; every thread gets its group's.  group < 0: contributes nothing
template <int RT>
__device__ __forceinline__ double2 group_sums(double a, double b, int group, int gs, double2* part) {
    // wave level first, group by group (a wave holds several groups), then the waves in LDS
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int g = 0; g < gs; ++g) {
        const double u = lane_group_sum(group == g ? a : 0.0, 64), v = lane_group_sum(group == g ? b : 0.0, 64);
        if (lane == 0) part[g * (RT / 64) + wave] = make_double2(u, v);
    }
    __syncthreads();
    double2 r = make_double2(0.0, 0.0);
    if (group >= 0)
#pragma unroll
        for (int w = 0; w < RT / 64; ++w) { const double2 v = part[group * (RT / 64) + w]; r.x += v.x; r.y += v.y; }
    return r;
}

template <typename T, int V, int ACT, int NR, int RT>
__global__ __launch_bounds__(RT, 4) void gn_resident_fwd_kernel(const NormArgs p, const Slab sl, int first_gap) {
    extern __shared__ double2 part[];                                      // [gs][waves]
    typedef typename PackedVec<T, V>::vec vec;
    if ((int)blockIdx.x >= first_gap) { zero_gaps<T>(p, first_gap); return; }
    int doc, c0;
    if (!slab_of(p, sl, doc, c0)) return;
    const int len = (int)p.len[doc];
    if (len <= 0) return;
    const int nx = sl.sc / V, ny = RT / nx, ry = threadIdx.x / nx, cx = threadIdx.x - ry * nx, cg = p.C / p.G;
    const bool on = ry < ny;
    const int64_t row0 = p.begin[doc];
    const T* x = reinterpret_cast<const T*>(p.x) + row0 * p.ldx + c0 + cx * V;
    T* y = reinterpret_cast<T*>(p.out) + row0 * p.C + c0 + cx * V;
    vec keep[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        const int r = k * ny + ry;
        if (on && r < len) keep[k] = *reinterpret_cast<const vec*>(x + (int64_t)r * p.ldx);
    }
    double s = 0.0, q = 0.0;
#pragma unroll
    for (int k = 0; k < NR; ++k)
        if (on && k * ny + ry < len)
#pragma unroll
            for (int i = 0; i < V; ++i) { const double d = (double)(float)keep[k][i]; s += d; q = fma(d, d, q); }
    for (int r = NR * ny + ry; on && r < len; r += ny) {
        float f[V];
        PackedVec<T, V>::load(f, x + (int64_t)r * p.ldx);
#pragma unroll
        for (int i = 0; i < V; ++i) { const double d = (double)f[i]; s += d; q = fma(d, d, q); }
    }
    const int g = on ? cx * V / cg : -1;
    const double2 t = group_sums<RT>(s, q, g, sl.gs, part);
    if (!on) return;
    const double count = (double)len * (double)cg, md = t.x / count, var = fmax(t.y / count - md * md, 0.0);
    const float m = (float)md, rs = (float)(1.0 / sqrt(var + (double)p.eps)), ml = (float)(md - (double)m);
    if (p.mean && ry == 0 && cx * V % cg == 0) {
        p.mean[(int64_t)doc * p.G + c0 / cg + g] = m;
        p.rstd[(int64_t)doc * p.G + c0 / cg + g] = rs;
        p.rest[(int64_t)doc * p.G + c0 / cg + g] = ml;
    }
    float w[V], b[V];
    PackedVec<float, V>::load(w, p.w + c0 + cx * V);
    PackedVec<float, V>::load(b, p.b + c0 + cx * V);
    auto apply = [&](float (&f)[V], int r) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = act_value<ACT, sizeof(T) == 4>(fmaf(centre<T>(f[i], m, ml) * rs, w[i], b[i]));
        PackedVec<T, V>::store(y + (int64_t)r * p.C, f);
    };
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        const int r = k * ny + ry;
        if (r < len) {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = (float)keep[k][i];
            apply(f, r);
        }
    }
    for (int r = NR * ny + ry; r < len; r += ny) {
        float f[V];
        PackedVec<T, V>::load(f, x + (int64_t)r * p.ldx);
        apply(f, r);
    }
}

template <typename T, int V, int ACT, int NR, int RT>
__global__ __launch_bounds__(RT, 4) void gn_resident_bwd_kernel(const NormArgs p, const Slab sl, int first_gap) {
    extern __shared__ double2 lds[];                                       // [gs][waves], then the channels' partial sums
    typedef typename PackedVec<T, V>::vec vec;
    if ((int)blockIdx.x >= first_gap) { if (p.out) zero_gaps<T>(p, first_gap); return; }
    int doc, c0;
    if (!slab_of(p, sl, doc, c0)) return;
    const int len = (int)p.len[doc];
    double2* sums = reinterpret_cast<double2*>(p.dsum) + (int64_t)doc * p.C + c0;
    if (len <= 0) {
        for (int c = threadIdx.x; c < sl.sc; c += RT) sums[c] = make_double2(0.0, 0.0);
        return;
    }
    const int nx = sl.sc / V, ny = RT / nx, ry = threadIdx.x / nx, cx = threadIdx.x - ry * nx, cg = p.C / p.G;
    const bool on = ry < ny;
    const int64_t row0 = p.begin[doc];
    const T* x = reinterpret_cast<const T*>(p.x) + row0 * p.ldx + c0 + cx * V;
    const T* dy = reinterpret_cast<const T*>(p.dy) + row0 * p.lddy + c0 + cx * V;
    vec kx[NR], kd[NR];
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        const int r = k * ny + ry;
        if (on && r < len) {
            kx[k] = *reinterpret_cast<const vec*>(x + (int64_t)r * p.ldx);
            kd[k] = *reinterpret_cast<const vec*>(dy + (int64_t)r * p.lddy);
        }
    }
    const int g = on ? cx * V / cg : -1;
    const int64_t stat = (int64_t)doc * p.G + c0 / cg + max(g, 0);
    const float m = p.mean[stat], rs = p.rstd[stat], ml = p.rest[stat];
    float w[V], b[V], s[V], q[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { const int c = c0 + min(cx, nx - 1) * V + i; w[i] = p.w[c]; b[i] = p.b[c]; s[i] = 0.f; q[i] = 0.f; }
    auto gather = [&](float xv, float dv, int i) {
        const float hat = centre<T>(xv, m, ml) * rs, dz = dv * act_slope<ACT, sizeof(T) == 4>(fmaf(hat, w[i], b[i]));
        s[i] += dz;
        q[i] = fmaf(dz, hat, q[i]);
    };
#pragma unroll
    for (int k = 0; k < NR; ++k)
        if (on && k * ny + ry < len)
#pragma unroll
            for (int i = 0; i < V; ++i) gather((float)kx[k][i], (float)kd[k][i], i);
    for (int r = NR * ny + ry; on && r < len; r += ny) {
        float f[V], d[V];
        PackedVec<T, V>::load(f, x + (int64_t)r * p.ldx);
        PackedVec<T, V>::load(d, dy + (int64_t)r * p.lddy);
#pragma unroll
        for (int i = 0; i < V; ++i) gather(f[i], d[i], i);
    }
    // channel sums: the threads' partials in LDS, added along the rows by RT / sc threads a channel, in two steps
    double2* part = lds;
    float2* stage = reinterpret_cast<float2*>(lds + sl.gs * (RT / 64));    // [ny][sc]
    if (on)
#pragma unroll
        for (int i = 0; i < V; ++i) stage[ry * sl.sc + cx * V + i] = make_float2(s[i], q[i]);
    __syncthreads();
    const int np = RT / sl.sc, pr = threadIdx.x / sl.sc, pc = threadIdx.x - pr * sl.sc;
    double sa = 0.0, sb = 0.0;
    if (pr < np)
        for (int r = pr; r < ny; r += np) { const float2 v = stage[r * sl.sc + pc]; sa += v.x; sb += v.y; }
    __syncthreads();
    double2* red = reinterpret_cast<double2*>(stage);                      // [np][sc]
    if (pr < np) red[pr * sl.sc + pc] = make_double2(sa, sb);
    __syncthreads();
    double ga = 0.0, gb = 0.0;
    int gg = -1;
    if ((int)threadIdx.x < sl.sc) {
        for (int i = 1; i < np; ++i) { const double2 v = red[i * sl.sc + threadIdx.x]; sa += v.x; sb += v.y; }
        sums[threadIdx.x] = make_double2(sa, sb);
        const double wc = (double)p.w[c0 + threadIdx.x];
        ga = wc * sa; gb = wc * sb;
        gg = (int)threadIdx.x / cg;
    }
    group_sums<RT>(ga, gb, gg, sl.gs, part);
    if (!on || !p.out) return;
    double2 t = make_double2(0.0, 0.0);
#pragma unroll
    for (int wv = 0; wv < RT / 64; ++wv) { const double2 v = part[g * (RT / 64) + wv]; t.x += v.x; t.y += v.y; }
    const double inv = 1.0 / ((double)len * (double)cg);
    const float c1 = (float)(t.x * inv), c2 = (float)(t.y * inv);
    T* dx = reinterpret_cast<T*>(p.out) + row0 * p.C + c0 + cx * V;
    auto apply = [&](float (&f)[V], const float (&d)[V], int r) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float hat = centre<T>(f[i], m, ml) * rs;
            const float gw = d[i] * act_slope<ACT, sizeof(T) == 4>(fmaf(hat, w[i], b[i])) * w[i];
            f[i] = rs * (gw - c1 - hat * c2);
        }
        PackedVec<T, V>::store(dx + (int64_t)r * p.C, f);
    };
#pragma unroll
    for (int k = 0; k < NR; ++k) {
        const int r = k * ny + ry;
        if (r < len) {
            float f[V], d[V];
#pragma unroll
            for (int i = 0; i < V; ++i) { f[i] = (float)kx[k][i]; d[i] = (float)kd[k][i]; }
            apply(f, d, r);
        }
    }
    for (int r = NR * ny + ry; r < len; r += ny) {
        float f[V], d[V];
        PackedVec<T, V>::load(f, x + (int64_t)r * p.ldx);
        PackedVec<T, V>::load(d, dy + (int64_t)r * p.lddy);
        apply(f, d, r);
    }
}

// dw, db: the documents' channel sums in their order, 64 channels a workgroup
__global__ __launch_bounds__(NTH) void gn_weight_sums_kernel(const NormArgs p) { weight_sums(p, (int)blockIdx.x * 64); }

// Slabs for documents of at most `longest` rows, vectors a thread keeps (0: such documents do not fit): whole groups, whole vectors in a group, the
// narrowest slab with 64 bytes of a row, narrower ones where only they fit.
int plan_slab(int64_t longest, int C, int G, int V, int RT, Slab& sl) {
    const int cg = C / G, max_nr = 7;
    if (cg % V || cg > RT) return 0;
    int gs = 1;
    while (gs < G && gs * cg * (16 / V) < 64) ++gs;
    while (G % gs) ++gs;
    for (;; gs = gs > 1 ? gs / 2 : 0) {
        if (!gs) return 0;
        if (G % gs) continue;
        const int sc = gs * cg;
        if (sc > RT) continue;
        const int ny = RT / (sc / V);
        const int64_t nr = cdiv(longest, ny);
        if (nr <= max_nr) { sl.gs = gs; sl.sc = sc; sl.nslab = G / gs; return (int)nr; }
    }
}

// parts of a tile: enough workgroups to fill the chip
int parts(int64_t M) { return M >= 65536 ? 1 : M >= 16384 ? 2 : 4; }

template <typename T, int V, int NR, int RT>
void resident(const NormArgs& p, const Slab& sl, int act, bool backward, hipStream_t s) {
    const int first_gap = (p.B * sl.nslab + 7) / 8 * 8;
    const dim3 grid((unsigned)(first_gap + GAP_WGS));
    const unsigned part = (unsigned)(sl.gs * (RT / 64) * sizeof(double2)), ny = (unsigned)(RT / (sl.sc / V));
    const unsigned stage = (unsigned)(ny * sl.sc * sizeof(float2)), red = (unsigned)(RT / sl.sc * sl.sc * sizeof(double2));
#define A(ACT_)                                                                                                                                 \
    if (!backward) hipLaunchKernelGGL((gn_resident_fwd_kernel<T, V, ACT_, NR, RT>), grid, dim3(RT), part, s, p, sl, first_gap);                      \
    else hipLaunchKernelGGL((gn_resident_bwd_kernel<T, V, ACT_, NR, RT>), grid, dim3(RT), part + (stage > red ? stage : red), s, p, sl, first_gap)
    if (act == ACT_RELU) { A(ACT_RELU); } else if (act == ACT_GELU) { A(ACT_GELU); } else if (act == ACT_SILU) { A(ACT_SILU); } else { A(ACT_NONE); }
#undef A
    if (backward && (p.dw || p.db)) hipLaunchKernelGGL(gn_weight_sums_kernel, dim3((unsigned)cdiv(p.C, 64)), dim3(NTH), 0, s, p);
}
template <typename T, int V>
bool try_resident(const NormArgs& p, int act, int64_t longest, bool backward, hipStream_t s) {
    if constexpr (V == 1) return false;
    else {
        Slab sl;
        if (!packed_aligned(p.w, 16) || !packed_aligned(p.b, 16)) return false;
        if ((int64_t)p.B * p.G > (int64_t)1 << 21) return false;             // (a launch has fewer than 2^32 threads)
        int nr = plan_slab(longest, p.C, p.G, V, 512, sl);
        if (nr == 0) {
            nr = plan_slab(longest, p.C, p.G, V, 1024, sl);
            if (nr == 0) return false;
            if (nr <= 5) resident<T, V, 5, 1024>(p, sl, act, backward, s); else resident<T, V, 7, 1024>(p, sl, act, backward, s);
        } else if (nr <= 2) resident<T, V, 2, 512>(p, sl, act, backward, s);
        else if (nr <= 4) resident<T, V, 4, 512>(p, sl, act, backward, s);
        else resident<T, V, 7, 512>(p, sl, act, backward, s);
        return true;
    }
}

template <typename T, int V>
void forward(NormArgs p, int act, int64_t longest, hipStream_t s) {
    if (try_resident<T, V>(p, act, longest, false, s)) return;
    const dim3 grid((unsigned)p.cap, (unsigned)p.sub);
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(NTH), (unsigned)((NTH * V + p.C) * sizeof(double2)), s, p);
    const bool direct = cdiv(longest, PACKED_TILE) * p.sub * p.G <= 2048;
    if (!direct) hipLaunchKernelGGL(gn_finish_kernel, dim3((unsigned)p.B), dim3(NTH), 0, s, p);
#define A(ACT_)                                                                                                                                 \
    if (direct) hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT_, true>), grid, dim3(NTH), (unsigned)(3 * p.G * sizeof(float)), s, p);             \
    else hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT_, false>), grid, dim3(NTH), 0, s, p)
    if (act == ACT_RELU) { A(ACT_RELU); } else if (act == ACT_GELU) { A(ACT_GELU); } else if (act == ACT_SILU) { A(ACT_SILU); } else { A(ACT_NONE); }
#undef A
}

template <typename T, int V>
void backward(NormArgs p, int act, int64_t longest, hipStream_t s) {
    if (try_resident<T, V>(p, act, longest, true, s)) return;
    const dim3 grid((unsigned)p.cap, (unsigned)p.sub), grid2((unsigned)(p.cap + cdiv(p.C, 64)), (unsigned)p.sub);
    const int cg = p.C / p.G, gchunk = cg >= 64 ? 1 : 64 / cg;
#define A(ACT_)                                                                                                                                 \
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, ACT_>), grid, dim3(NTH), 0, s, p);                                                              \
    hipLaunchKernelGGL(gn_bwd_docs_kernel, dim3((unsigned)p.B, (unsigned)cdiv(p.G, gchunk)), dim3(512), (unsigned)(gchunk * cg * sizeof(double2)), s, p, gchunk); \
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT_>), grid2, dim3(NTH), 0, s, p)
    if (act == ACT_RELU) { A(ACT_RELU); } else if (act == ACT_GELU) { A(ACT_GELU); } else if (act == ACT_SILU) { A(ACT_SILU); } else { A(ACT_NONE); }
#undef A
}

}  // namespace

// Bytes of the workspace of one call (forward or backward).
extern "C" int64_t osp_group_norm_workspace_bytes(int64_t B, int64_t M, int64_t C, int64_t G, int64_t backward) {
    if (B <= 0 || M < 0 || C <= 0 || G <= 0) return 0;
    const int64_t slots = (M / PACKED_TILE + B) * parts(M);
    if (!backward) return slots * G * 16 + 256;
    return slots * C * 8 + B * C * 16 + B * G * 8 + 512;
}

extern "C" int osp_group_norm_fwd(const void* x, int64_t ldx, int64_t bf16, const float* w, const float* b, void* y, float* stats,
                                  void* workspace, const int64_t* begin, const int64_t* len, const int32_t* base, const int32_t* tiles, const int32_t* ntiles,
                                  int64_t cap, int64_t B, int64_t M, int64_t longest, int64_t C, int64_t G, float eps, int64_t act,
                                  hipStream_t stream) {
    OSP_CHECK_ARG(x && w && b && y && stats && workspace && begin && len && base && tiles && ntiles, "null pointer");
    OSP_CHECK_ARG(B > 0 && M > 0 && longest > 0 && C > 0 && C <= MAXC && G > 0 && C % G == 0 && ldx >= C, "channels (at most 2048) must be a multiple of groups");
    OSP_CHECK_ARG(eps > 0.f && act >= ACT_NONE && act <= ACT_SILU && cap > 0 && cap < (int64_t)1 << 30 && packed_aligned(workspace, 16), "bad eps, activation or workspace");
    NormArgs p = {};
    p.x = x; p.ldx = ldx; p.w = w; p.b = b; p.out = y; p.mean = stats; p.rstd = stats + B * G; p.rest = stats + 2 * B * G; p.part = reinterpret_cast<double*>(workspace);
    p.begin = begin; p.len = len; p.base = base; p.tiles = reinterpret_cast<const PackedTile*>(tiles); p.ntiles = ntiles;
    p.B = (int)B; p.C = (int)C; p.G = (int)G; p.cap = (int)cap; p.sub = parts(M); p.eps = eps;
    const int V = bf16 ? 8 : 4;
    const bool wide = C % V == 0 && ldx % V == 0 && packed_aligned(x, 16) && packed_aligned(y, 16);
    if (bf16) { if (wide) forward<__bf16, 8>(p, (int)act, longest, stream); else forward<__bf16, 1>(p, (int)act, longest, stream); }
    else { if (wide) forward<float, 4>(p, (int)act, longest, stream); else forward<float, 1>(p, (int)act, longest, stream); }
    OSP_LAUNCH_CHECK();
    return OSP_OK;
}

extern "C" int osp_group_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t bf16, const float* w, const float* b,
                                  const float* stats, void* dx, float* dw, int64_t add_w, float* db, int64_t add_b, void* workspace,
                                  const int64_t* begin, const int64_t* len, const int32_t* base, const int32_t* tiles, const int32_t* ntiles,
                                  int64_t cap, int64_t B, int64_t M, int64_t longest, int64_t C, int64_t G, int64_t act, hipStream_t stream) {
    OSP_CHECK_ARG(dy && x && w && b && stats && workspace && begin && len && base && tiles && ntiles, "null pointer");
    OSP_CHECK_ARG(B > 0 && M > 0 && longest > 0 && C > 0 && C <= MAXC && G > 0 && C % G == 0 && ldx >= C && lddy >= C, "channels (at most 2048) must be a multiple of groups");
    OSP_CHECK_ARG(act >= ACT_NONE && act <= ACT_SILU && cap > 0 && cap < (int64_t)1 << 30 && packed_aligned(workspace, 16), "bad activation or workspace");
    NormArgs p = {};
    p.x = x; p.ldx = ldx; p.dy = dy; p.lddy = lddy; p.w = w; p.b = b; p.out = dx;
    p.mean = const_cast<float*>(stats); p.rstd = p.mean + B * G; p.rest = p.mean + 2 * B * G; p.dw = dw; p.db = db; p.add_w = (int)(add_w != 0); p.add_b = (int)(add_b != 0);
    p.begin = begin; p.len = len; p.base = base; p.tiles = reinterpret_cast<const PackedTile*>(tiles); p.ntiles = ntiles;
    p.B = (int)B; p.C = (int)C; p.G = (int)G; p.cap = (int)cap; p.sub = parts(M);
    const int64_t slots = (M / PACKED_TILE + B) * p.sub;
    char* ws = reinterpret_cast<char*>(workspace);
    p.dsum = reinterpret_cast<double*>(ws);                            // (B, C, 2) f64
    p.cpart = reinterpret_cast<float*>(ws + B * C * 16);               // (slots, C, 2) f32
    p.coef = reinterpret_cast<float*>(ws + B * C * 16 + slots * C * 8);
    const int V = bf16 ? 8 : 4;
    const bool wide = C % V == 0 && ldx % V == 0 && lddy % V == 0 && packed_aligned(x, 16) && packed_aligned(dy, 16) && packed_aligned(dx, 16);
    if (bf16) { if (wide) backward<__bf16, 8>(p, (int)act, longest, stream); else backward<__bf16, 1>(p, (int)act, longest, stream); }
    else { if (wide) backward<float, 4>(p, (int)act, longest, stream); else backward<float, 1>(p, (int)act, longest, stream); }
    OSP_LAUNCH_CHECK();
    return OSP_OK;
}
