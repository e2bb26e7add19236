// What the packed-row operators share (attention over documents, rotary positions, group norm): the tile list of a batch.
//
// A batch is a table of M rows.  Document b owns the rows [begin[b], begin[b] + len[b]); rows of no document (a padded tail, the rows behind
// the last offset) are written as zeros by every operator.  Both live in device memory, so that no operator needs the lengths on the
// host: osp_packed_rows_plan turns offsets or lengths into begin / len and into a list of tiles of PACKED_TILE rows, and a workgroup reads its
// tile from the list.  The grid is the host's upper bound on the list; workgroups behind its end leave at once.
#pragma once
#include "osp_common.h"

#define PACKED_TILE 128

struct PackedTile {          // 16 bytes, one load
    int doc;                 // -1: rows of no document
    int row0;                // first row of the tile in the table
    int n;                   // rows (1 .. PACKED_TILE)
    int i0;                  // index of the first row inside its document (a multiple of PACKED_TILE)
};

typedef __bf16 pk_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pk_bf16x4 __attribute__((ext_vector_type(4)));

// V consecutive elements <-> f32 registers; V * sizeof(T) is 4, 8 or 16 bytes (or one element), the address aligned to it
template <typename T, int V>
struct PackedVec {
    typedef T vec __attribute__((ext_vector_type(V)));
    static __device__ __forceinline__ void load(float (&f)[V], const T* p) {
        const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (float)v[i];
    }
    static __device__ __forceinline__ void store(T* p, const float (&f)[V]) {
        vec v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)f[i];              // round to nearest even: the operator's one rounding to the output's type
        *reinterpret_cast<vec*>(p) = v;
    }
};
template <typename T>
struct PackedVec<T, 1> {
    static __device__ __forceinline__ void load(float (&f)[1], const T* p) { f[0] = (float)*p; }
    static __device__ __forceinline__ void store(T* p, const float (&f)[1]) { *p = (T)f[0]; }
};

static inline bool packed_aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }
