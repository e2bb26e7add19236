// Rotary positions on packed rows: every head of q and k turned pair by pair, one launch for both, forward and backward.
//   pos   = first[doc] + index of the row in its document,   angle_i = pos f_i,   i < R / 2
//   (a, b) -> mag (a cos - b sin, a sin + b cos)             pairs (2 i, 2 i + 1): interleaved;  (i, i + R / 2): half
//   backward: the transpose, mag (a cos + b sin, -a sin + b cos), on the incoming gradients; channels R .. D - 1 pass unchanged
//
// The angle is formed in 64 bits: at position 10^6 a 32-bit product is off by 0.06 rad.  The caller hands f_i / (2 pi) ("turns per
// position"); the product's nearest quarter turn is taken off in 64 bits and the rest, |r| <= 1/8 turn, goes to f32: an angle of at most
// pi / 4 whose rounding is 2^-25 of it.  sin and cos of it are Taylor sums (degree 9 and 10; the first term left out is below 2e-9).
//
// Bound: HBM.  A thread owns V pairs of one row and keeps their cos / sin in registers over all heads of q and k, so the 64-bit work is done
// once per row and not once per head; all its loads and stores are 16 bytes where alignment allows.
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

// V pairs per slot.  Slots of a row: R / 2 / V that turn, then (D - R) / (2 V) rounded up that copy (2 V channels each, the last one short).
template <typename TI, typename TO, int V, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs p, int rows_per_wg) {
    const int nt = p.ntiles[1];
    if ((int)blockIdx.x >= nt) return;
    const PackedTile tile = p.tiles[blockIdx.x];
    const int turning = p.R / 2 / V, copying = (p.D - p.R + 2 * V - 1) / (2 * V), slots = turning + copying;
    const int r_lo = blockIdx.y * rows_per_wg, r_hi = min(tile.n, r_lo + rows_per_wg);
    if (r_lo >= r_hi) return;
    const int total = (r_hi - r_lo) * slots;
    if (tile.doc < 0) {                                           // rows of no document: zeros
        for (int which = 0; which < 2; ++which) {
            TO* y = reinterpret_cast<TO*>(p.y[which]) + (int64_t)(tile.row0 + r_lo) * p.heads[which] * p.D;
            const int64_t n = (int64_t)(r_hi - r_lo) * p.heads[which] * p.D;
            for (int64_t i = threadIdx.x; i < n; i += 256) y[i] = (TO)0.f;
        }
        return;
    }
    const int64_t first = p.first ? p.first[tile.doc] : 0;
    for (int u = threadIdx.x; u < total; u += 256) {
        const int r = r_lo + u / slots, slot = u % slots;
        const int64_t row = (int64_t)tile.row0 + r;
        if (slot < turning) {
            const double pos = (double)(first + tile.i0 + r);
            float s[V], c[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                turn_sincos(pos * p.turns[slot * V + i], s[i], c[i]);
                s[i] *= p.inverse ? -p.mag : p.mag;
                c[i] *= p.mag;
            }
            for (int which = 0; which < 2; ++which) {
                const TI* x = reinterpret_cast<const TI*>(p.x[which]) + row * p.xr[which];
                TO* y = reinterpret_cast<TO*>(p.y[which]) + row * p.heads[which] * p.D;
#pragma unroll 4
                for (int h = 0; h < p.heads[which]; ++h) {
                    if constexpr (HALF) {
                        const int at = slot * V;
                        float a[V], b[V], ya[V], yb[V];
                        PackedVec<TI, V>::load(a, x + h * p.xh[which] + at);
                        PackedVec<TI, V>::load(b, x + h * p.xh[which] + p.R / 2 + at);
#pragma unroll
                        for (int i = 0; i < V; ++i) { ya[i] = a[i] * c[i] - b[i] * s[i]; yb[i] = a[i] * s[i] + b[i] * c[i]; }
                        PackedVec<TO, V>::store(y + h * p.D + at, ya);
                        PackedVec<TO, V>::store(y + h * p.D + p.R / 2 + at, yb);
                    } else {
                        const int at = slot * 2 * V;
                        float a[2 * V], b[2 * V];
                        PackedVec<TI, 2 * V>::load(a, x + h * p.xh[which] + at);
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            b[2 * i] = a[2 * i] * c[i] - a[2 * i + 1] * s[i];
                            b[2 * i + 1] = a[2 * i] * s[i] + a[2 * i + 1] * c[i];
                        }
                        PackedVec<TO, 2 * V>::store(y + h * p.D + at, b);
                    }
                }
            }
        } else {
            const int at = p.R + (slot - turning) * 2 * V, n = min(2 * V, p.D - at);
            for (int which = 0; which < 2; ++which) {
                const TI* x = reinterpret_cast<const TI*>(p.x[which]) + row * p.xr[which] + at;
                TO* y = reinterpret_cast<TO*>(p.y[which]) + row * p.heads[which] * p.D + at;
                for (int h = 0; h < p.heads[which]; ++h)
                    for (int i = 0; i < n; ++i) y[h * p.D + i] = (TO)(float)x[h * p.xh[which] + i];
            }
        }
    }
}

template <typename TI, typename TO, bool HALF>
void launch(const RotaryArgs& p, int V, dim3 grid, int rows_per_wg, hipStream_t stream) {
    // V pairs: the widest accesses of 16 bytes that alignment and R allow (one pair otherwise)
    constexpr int VW = HALF ? (sizeof(TI) == 2 ? 8 : 4) : (sizeof(TI) == 2 ? 4 : 2);
    if (V > 1) hipLaunchKernelGGL((rotary_kernel<TI, TO, VW, HALF>), grid, dim3(256), 0, stream, p, rows_per_wg);
    else hipLaunchKernelGGL((rotary_kernel<TI, TO, 1, HALF>), grid, dim3(256), 0, stream, p, rows_per_wg);
}

}  // namespace

extern "C" int osp_rotary(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, int64_t in_bf16,
                          void* qo, void* ko, int64_t out_bf16, const double* turns, const int32_t* tiles, const int32_t* ntiles, int64_t cap,
                          const int64_t* first, int64_t Hq, int64_t Hk, int64_t D, int64_t R, int64_t interleaved, float mag,
                          int64_t inverse, hipStream_t stream) {
    OSP_CHECK_ARG(q && k && qo && ko && turns && tiles && ntiles, "null pointer");
    OSP_CHECK_ARG(cap > 0 && cap < (int64_t)1 << 31 && Hq > 0 && Hk > 0 && Hq <= 65536 && Hk <= 65536, "bad tile list or head counts");
    OSP_CHECK_ARG(D > 0 && D <= 8192 && R >= 2 && R <= D && R % 2 == 0, "an even number of turned channels, at most the head's");
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
    const int slots = (int)(R / 2 / V + (D - R + 2 * V - 1) / (2 * V));
    // rows of a workgroup: about one slot per thread
    int rows = 256 / slots;
    rows = rows < 1 ? 1 : rows > PACKED_TILE ? PACKED_TILE : rows;
    const dim3 grid((unsigned)cap, (unsigned)cdiv(PACKED_TILE, rows));
    if (in_bf16 && out_bf16) { if (interleaved) launch<__bf16, __bf16, false>(p, V, grid, rows, stream); else launch<__bf16, __bf16, true>(p, V, grid, rows, stream); }
    else if (in_bf16) { if (interleaved) launch<__bf16, float, false>(p, V, grid, rows, stream); else launch<__bf16, float, true>(p, V, grid, rows, stream); }
    else if (out_bf16) { if (interleaved) launch<float, __bf16, false>(p, V, grid, rows, stream); else launch<float, __bf16, true>(p, V, grid, rows, stream); }
    else { if (interleaved) launch<float, float, false>(p, V, grid, rows, stream); else launch<float, float, true>(p, V, grid, rows, stream); }
    OSP_LAUNCH_CHECK();
    return OSP_OK;
}
