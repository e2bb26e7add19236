// Rotary positions on packed rows: every head of q and k turned pair by pair, one launch for both, forward and backward.
//   pos   = first[doc] + index of the row in its document,   angle_i = pos f_i,   i < R / 2
//   (a, b) -> mag (a cos - b sin, a sin + b cos)             pairs (2 i, 2 i + 1): interleaved;  (i, i + R / 2): half
//   backward: the transpose, mag (a cos + b sin, -a sin + b cos), on the incoming gradients; channels R .. D - 1 pass unchanged
//
// The angle is formed in 64 bits: at position 10^6 a 32-bit product is off by 0.06 rad.  The caller hands f_i / (2 pi) ("turns per
// position"); the product's nearest quarter turn is taken off in 64 bits and the rest, |r| <= 1/8 turn, goes to f32: an angle of at most
// pi / 4 whose rounding is 2^-25 of it.  sin and cos of it are Taylor sums (degree 9 and 10; the first term left out is below 2e-9).
//
// Bound: HBM.  The 64-bit work is done once per row and pair, into LDS, and serves all heads of q and k; the heads are then walked in the order of memory
// with accesses of 16 bytes where alignment allows.  (A thread that kept its pairs' cos and sin in registers and walked the heads itself read every row
// in strides of a head: 87 us where this takes 75.)
//
// Measured: 24 k rows, 16 + 4 heads of 128, bf16: 75 us, 4.4 TB/s (a copy reaches 5.1);  17 k rows, 4 + 4 heads of 64, half of each turned, f32: 15.1 us, 4.8 TB/s;
// 8 rows: 4.7 us, latency.
#include "packed_common.h"

namespace {

struct RotaryArgs {
    const void* x[2];                     // q, k
    void* y[2];
    int64_t xr[2], xh[2];                 // row and head stride of the inputs (elements); outputs are (M, heads, D) contiguous
    int heads[2];
    const double* turns;                  // R / 2
    const PackedTile* tiles;
    const int* ntiles;
    const int64_t* first;                 // per document, or null
    int D, R;
    float mag;
    int inverse;
};

__device__ __forceinline__ void turn_sincos(double t, float& s, float& c) {
    t -= rint(t);                                                 // whole turns
    const double quarter = rint(4.0 * t);
    const float a = (float)((t - 0.25 * quarter) * 6.283185307179586476925);
    const float z = a * a;
    float sn = fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f);
    sn = fmaf(a * z, sn, a);                                      // a - a^3/3! + a^5/5! - a^7/7! + a^9/9!
    float cs = fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f);
    cs = fmaf(z * z, cs, fmaf(z, -0.5f, 1.0f));                   // 1 - a^2/2! + a^4/4! - a^6/6! + a^8/8! - a^10/10!
    const int k = (int)quarter & 3;
    const float s1 = (k & 1) ? cs : sn, c1 = (k & 1) ? sn : cs;
    s = (k & 2) ? -s1 : s1;
    c = ((k + 1) & 2) ? -c1 : c1;
}

// V pairs per slot.  First the workgroup's rows' cos and sin go to LDS (rows x R / 2 pairs, mag and the direction's sign included); then its threads walk
// (row, head, slot) in the order of memory, BATCH vectors in flight each.
template <typename TI, typename TO, int V, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs p, int rows_per_wg) {
    extern __shared__ float2 turn_l[];
    constexpr int BATCH = 4, W = HALF ? V : 2 * V;                 // channels of one access
    const PackedTile tile = p.tiles[blockIdx.x];
    if ((int)blockIdx.x >= p.ntiles[1]) return;
    const int r_lo = blockIdx.y * rows_per_wg, n = min(tile.n - r_lo, rows_per_wg), tid = threadIdx.x;
    if (n <= 0) return;
    const int64_t row0 = (int64_t)tile.row0 + r_lo;
    if (tile.doc < 0) {                                           // rows of no document: zeros
        for (int which = 0; which < 2; ++which) {
            TO* y = reinterpret_cast<TO*>(p.y[which]) + row0 * p.heads[which] * p.D;
            const int64_t total = (int64_t)n * p.heads[which] * p.D;
            for (int64_t i = tid; i < total; i += 256) y[i] = (TO)0.f;
        }
        return;
    }
    const int half = p.R / 2;
    const int64_t pos0 = (p.first ? p.first[tile.doc] : 0) + tile.i0 + r_lo;
    for (int u = tid; u < n * half; u += 256) {
        const int r = u / half;
        float s, c;
        turn_sincos((double)(pos0 + r) * p.turns[u - r * half], s, c);
        turn_l[u] = make_float2(c * p.mag, p.inverse ? -s * p.mag : s * p.mag);
    }
    __syncthreads();
    const int turning = half / V, lanes = min(turning, 256), step = 256 / lanes, slot0 = tid % lanes, item0 = tid / lanes;
    for (int which = 0; which < 2; ++which) {
        const int heads = p.heads[which], items = n * heads;
        const TI* x = reinterpret_cast<const TI*>(p.x[which]) + row0 * p.xr[which];
        TO* y = reinterpret_cast<TO*>(p.y[which]) + row0 * heads * p.D;
        for (int slot = slot0; slot < turning && item0 < step; slot += lanes) {
            const int at = slot * W;
            for (int item = item0; item < items; item += BATCH * step) {
                float a[BATCH][W], b[BATCH][HALF ? W : 1];
                int rr[BATCH];
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const int it = item + j * step;
                    rr[j] = it / heads;
                    if (it < items) {
                        const TI* src = x + rr[j] * p.xr[which] + (it - rr[j] * heads) * p.xh[which] + at;
                        PackedVec<TI, W>::load(a[j], src);
                        if constexpr (HALF) PackedVec<TI, W>::load(b[j], src + half);
                    }
                }
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    const int it = item + j * step;
                    if (it >= items) continue;
                    const float2* cs = turn_l + rr[j] * half + slot * V;
                    TO* dst = y + (int64_t)it * p.D + at;
                    float u[W], w[HALF ? W : 1];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float2 t = cs[i];
                        if constexpr (HALF) { u[i] = a[j][i] * t.x - b[j][i] * t.y; w[i] = a[j][i] * t.y + b[j][i] * t.x; }
                        else { u[2 * i] = a[j][2 * i] * t.x - a[j][2 * i + 1] * t.y; u[2 * i + 1] = a[j][2 * i] * t.y + a[j][2 * i + 1] * t.x; }
                    }
                    PackedVec<TO, W>::store(dst, u);
                    if constexpr (HALF) PackedVec<TO, W>::store(dst + half, w);
                }
            }
        }
        const int rest = p.D - p.R;                               // the remaining channels pass
        if (rest) {
            const int per = V > 1 && rest % W == 0 ? W : 1, chunks = rest / per;
            for (int u = tid; u < items * chunks; u += 256) {
                const int it = u / chunks, c = p.R + (u - it * chunks) * per, r = it / heads;
                const TI* src = x + r * p.xr[which] + (it - r * heads) * p.xh[which] + c;
                TO* dst = y + (int64_t)it * p.D + c;
                if (per > 1) { float f[W]; PackedVec<TI, W>::load(f, src); PackedVec<TO, W>::store(dst, f); }
                else *dst = (TO)(float)*src;
            }
        }
    }
}

template <typename TI, typename TO, bool HALF>
void launch(const RotaryArgs& p, int V, dim3 grid, int rows_per_wg, hipStream_t stream) {
    // V pairs: the widest accesses of 16 bytes that alignment and R allow (one pair otherwise)
    constexpr int VW = HALF ? (sizeof(TI) == 2 ? 8 : 4) : (sizeof(TI) == 2 ? 4 : 2);
    if (V > 1) hipLaunchKernelGGL((rotary_kernel<TI, TO, VW, HALF>), grid, dim3(256), (unsigned)(rows_per_wg * p.R * 4), stream, p, rows_per_wg);
    else hipLaunchKernelGGL((rotary_kernel<TI, TO, 1, HALF>), grid, dim3(256), (unsigned)(rows_per_wg * p.R * 4), stream, p, rows_per_wg);
}

}  // namespace

extern "C" int osp_rotary(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, int64_t in_bf16,
                          void* qo, void* ko, int64_t out_bf16, const double* turns, const int32_t* tiles, const int32_t* ntiles, int64_t cap,
                          const int64_t* first, int64_t Hq, int64_t Hk, int64_t D, int64_t R, int64_t interleaved, float mag,
                          int64_t inverse, hipStream_t stream) {
    OSP_CHECK_ARG(q && k && qo && ko && turns && tiles && ntiles, "null pointer");
    OSP_CHECK_ARG(cap > 0 && cap < (int64_t)1 << 31 && Hq > 0 && Hk > 0 && Hq <= 65536 && Hk <= 65536, "bad tile list or head counts");
    OSP_CHECK_ARG(D > 0 && D <= 8192 && R >= 2 && R <= D && R % 2 == 0, "an even number of turned channels, at most the head's");
    OSP_CHECK_ARG(Hq * D <= 1 << 26 && Hk * D <= 1 << 26, "a row has at most 2^26 channels");
    RotaryArgs p;
    p.x[0] = q; p.x[1] = k; p.y[0] = qo; p.y[1] = ko;
    p.xr[0] = q_row; p.xr[1] = k_row; p.xh[0] = q_head; p.xh[1] = k_head;
    p.heads[0] = (int)Hq; p.heads[1] = (int)Hk;
    p.turns = turns; p.tiles = reinterpret_cast<const PackedTile*>(tiles); p.ntiles = ntiles; p.first = first;
    p.D = (int)D; p.R = (int)R; p.mag = mag; p.inverse = (int)(inverse != 0);
    const int esz = in_bf16 ? 2 : 4, osz = out_bf16 ? 2 : 4;
    const int VW = interleaved ? (in_bf16 ? 4 : 2) : (in_bf16 ? 8 : 4);
    const int run = interleaved ? 2 * VW : VW;                     // consecutive channels of one access
    bool wide = R % (2 * VW) == 0 && D % run == 0 && (interleaved || (R / 2) % VW == 0);
    const int64_t ib = (int64_t)run * esz, ob = (int64_t)run * osz < 16 ? (int64_t)run * osz : 16;
    for (int w = 0; w < 2; ++w)
        wide = wide && packed_aligned(p.x[w], ib) && packed_aligned(p.y[w], ob) && p.xr[w] % run == 0 && p.xh[w] % run == 0;
    const int V = wide ? VW : 1;
    // rows of a workgroup: 16, fewer where their cos and sin would take more than 32 KB
    int rows = (int)(8192 / R);
    rows = rows < 1 ? 1 : rows > 16 ? 16 : rows;
    const dim3 grid((unsigned)cap, (unsigned)cdiv(PACKED_TILE, rows));
    if (in_bf16 && out_bf16) { if (interleaved) launch<__bf16, __bf16, false>(p, V, grid, rows, stream); else launch<__bf16, __bf16, true>(p, V, grid, rows, stream); }
    else if (in_bf16) { if (interleaved) launch<__bf16, float, false>(p, V, grid, rows, stream); else launch<__bf16, float, true>(p, V, grid, rows, stream); }
    else if (out_bf16) { if (interleaved) launch<float, __bf16, false>(p, V, grid, rows, stream); else launch<float, __bf16, true>(p, V, grid, rows, stream); }
    else { if (interleaved) launch<float, float, false>(p, V, grid, rows, stream); else launch<float, float, true>(p, V, grid, rows, stream); }
    OSP_LAUNCH_CHECK();
    return OSP_OK;
}
