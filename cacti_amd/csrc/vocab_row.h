// A row of the vocabulary's width at any address, read in 16-byte pieces: piece c has the elements 8 c - off .. 8 c - off + 7,
// off being how far the row begins behind a 16-byte boundary.
#pragma once
#include "common.h"

namespace cacti {

struct VocabRow {
    const half_t *row;
    int V, off;
    __device__ __forceinline__ VocabRow(const half_t *r, int v) : row(r), V(v), off((int)(reinterpret_cast<uintptr_t>(r) / 2 & 7)) {}
    __device__ __forceinline__ int pieces() const { return (V + off + 7) / 8; }
    __device__ __forceinline__ int first(int c) const { return 8 * c - off; }
    __device__ __forceinline__ bool whole(int c) const { return first(c) >= 0 && first(c) + 8 <= V; }
    // elements beside the row are `pad`
    __device__ __forceinline__ h8 load(int c, half_t pad) const
    {
        const int j = first(c);
        if (whole(c)) return ld8(row + j);
        h8 x;
#pragma unroll
        for (int k = 0; k < 8; k++) x.v[k] = j + k >= 0 && j + k < V ? row[j + k] : pad;
        return x;
    }
};

}  // namespace cacti
