// Documents of a packed batch -> begin / len per document, the slot of its first tile, and the tile list the packed-row operators walk.
// One workgroup: B documents are a few thousand at most, and the list is some thousand entries of 16 bytes.  A batch builds it once and every
// layer and direction uses it.
//
// Offsets that fall outside [0, M] are clamped and an offset below its predecessor counts as its predecessor (running maximum): whatever
// the table holds, documents are disjoint row ranges inside the batch and no operator reads or writes outside it.
//
// Tiles stand in the list by descending index inside their document: under a causal mask a late query tile has the most keys, so the
// longest workgroups start first.  The order inside one index is that of LDS atomics; it decides only when a tile is computed.
#include "packed_common.h"

namespace {
constexpr int NT = 1024, NBIN = 1024;

__device__ __forceinline__ int64_t wave_scan_max(int64_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(v, o, 64);
        if (lane >= o && u > v) v = u;
    }
    return v;
}
__device__ __forceinline__ int wave_scan_sum(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}
}  // namespace

__global__ __launch_bounds__(NT) void packed_rows_plan_kernel(const int64_t* __restrict__ src, int padded, int64_t B, int64_t M, int64_t T,
                                                              int64_t* __restrict__ begin, int64_t* __restrict__ len, int* __restrict__ base,
                                                              PackedTile* __restrict__ tiles, int* __restrict__ ntiles, int cap) {
    __shared__ int64_t wmax[16];
    __shared__ int wsum[16];
    __shared__ int bins[NBIN];
    __shared__ int n_gap;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < NBIN; i += NT) bins[i] = 0;
    if (tid == 0) n_gap = 0;
    int64_t carry_max = 0;
    int carry_sum = 0;
    for (int64_t b0 = 0; b0 < B; b0 += NT) {
        const int64_t b = b0 + tid;
        int64_t bg = 0, ln = 0;
        if (padded) {
            if (b < B) { bg = b * T; ln = min(max(src[b], (int64_t)0), T); }
        } else {
            int64_t e = 0, e1 = 0;
            if (b < B) { e = min(max(src[b], (int64_t)0), M); e1 = min(max(src[b + 1], (int64_t)0), M); }
            int64_t v = wave_scan_max(e, lane);
            if (lane == 63) wmax[wave] = v;
            __syncthreads();
            int64_t pre = carry_max;
            for (int w = 0; w < wave; ++w) pre = max(pre, wmax[w]);
            int64_t all = carry_max;
            for (int w = 0; w < NT / 64; ++w) all = max(all, wmax[w]);
            bg = max(v, pre);
            ln = max(e1 - bg, (int64_t)0);
            carry_max = all;
        }
        if (b >= B) ln = 0;
        const int nt = (int)((ln + PACKED_TILE - 1) / PACKED_TILE);
        int s = wave_scan_sum(nt, lane);
        if (lane == 63) wsum[wave] = s;
        __syncthreads();
        int pre = carry_sum, all = carry_sum;
        for (int w = 0; w < NT / 64; ++w) { if (w < wave) pre += wsum[w]; all += wsum[w]; }
        if (b < B) { begin[b] = bg; len[b] = ln; base[b] = pre + s - nt; }
        carry_sum = all;
        __syncthreads();                                          // wmax / wsum are reused; begin / len visible to the whole workgroup below
    }
    __threadfence_block();
    __syncthreads();
    for (int64_t b = wave; b < B; b += NT / 64) {                 // one wave per document, lanes over its tiles
        const int nt = (int)((len[b] + PACKED_TILE - 1) / PACKED_TILE);
        for (int t = lane; t < nt; t += 64) atomicAdd(&bins[NBIN - 1 - min(t, NBIN - 1)], 1);
    }
    __syncthreads();
    {                                                             // exclusive scan of the bins (one per thread)
        const int own = bins[tid];
        const int s = wave_scan_sum(own, lane);
        if (lane == 63) wsum[wave] = s;
        __syncthreads();
        int pre = 0;
        for (int w = 0; w < wave; ++w) pre += wsum[w];
        bins[tid] = pre + s - own;
    }
    __syncthreads();
    const int ndoc = carry_sum;
    for (int64_t b = wave; b < B; b += NT / 64) {
        const int64_t ln = len[b], bg = begin[b];
        const int nt = (int)((ln + PACKED_TILE - 1) / PACKED_TILE);
        for (int t = lane; t < nt; t += 64) {
            const int slot = atomicAdd(&bins[NBIN - 1 - min(t, NBIN - 1)], 1);
            if (slot < cap)
                tiles[slot] = PackedTile{(int)b, (int)(bg + (int64_t)t * PACKED_TILE), (int)min((int64_t)PACKED_TILE, ln - (int64_t)t * PACKED_TILE), t * PACKED_TILE};
        }
        // rows of no document: behind this document up to the next one's first row (or its padded end / the end of the table)
        const int64_t g0 = bg + ln, g1 = padded ? (b + 1) * T : (b + 1 < B ? begin[b + 1] : M);
        const int64_t h1 = (b == 0 && !padded) ? bg : 0;          // and in front of the first document
        for (int64_t r = g0 + (int64_t)lane * PACKED_TILE; r < g1; r += 64 * PACKED_TILE) {
            const int slot = ndoc + atomicAdd(&n_gap, 1);
            if (slot < cap) tiles[slot] = PackedTile{-1, (int)r, (int)min((int64_t)PACKED_TILE, g1 - r), 0};
        }
        for (int64_t r = (int64_t)lane * PACKED_TILE; r < h1; r += 64 * PACKED_TILE) {
            const int slot = ndoc + atomicAdd(&n_gap, 1);
            if (slot < cap) tiles[slot] = PackedTile{-1, (int)r, (int)min((int64_t)PACKED_TILE, h1 - r), 0};
        }
    }
    __syncthreads();
    if (tid == 0) { ntiles[0] = min(ndoc, cap); ntiles[1] = min(ndoc + n_gap, cap); }
}

// Most tiles a batch can have: documents cut M rows into at most M / PACKED_TILE + B pieces (each document ends with at most one short tile);
// rows of no document stand in front, between or behind (decreasing offsets leave them anywhere), or once per padded document.
extern "C" int64_t osp_packed_rows_tiles(int64_t B, int64_t M) {
    if (B <= 0 || M < 0) return 0;
    return M / PACKED_TILE + 2 * B + 2;
}

extern "C" int osp_packed_rows_plan(const int64_t* src, int64_t padded, int64_t B, int64_t M, int64_t T, int64_t* begin, int64_t* len,
                                    int32_t* base, int32_t* tiles, int32_t* ntiles, int64_t cap, hipStream_t stream) {
    OSP_CHECK_ARG(src && begin && len && base && tiles && ntiles && B > 0 && M >= 0, "bad args");
    // (row numbers are 32-bit in the kernels, which look up to a few tiles beyond a row)
    OSP_CHECK_ARG(M <= ((int64_t)1 << 31) - 65536 && B < (int64_t)1 << 24, "at most 2^31 - 65536 rows and 2^24 - 1 documents");
    OSP_CHECK_ARG(!padded || (T >= 0 && T * B == M), "a padded batch has B * T rows");
    OSP_CHECK_ARG(cap >= osp_packed_rows_tiles(B, M), "tile list shorter than osp_packed_rows_tiles(B, M)");
    OSP_CHECK_ARG(packed_aligned(tiles, 16), "tile list must be 16-byte aligned");
    hipLaunchKernelGGL(packed_rows_plan_kernel, dim3(1), dim3(NT), 0, stream, src, (int)(padded != 0), B, M, T, begin, len, base,
                       reinterpret_cast<PackedTile*>(tiles), ntiles, (int)cap);
    OSP_LAUNCH_CHECK();
    return OSP_OK;
}
