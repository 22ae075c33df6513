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

// A row of up to 8 T NP + 7 elements, held by T threads: of its whole 16-byte pieces those lo + tid + i T, and of up to 14
// elements beside them one for each of the first threads.  (The pieces may be those of another row: loads of 16 bytes may begin
// at any element.)
typedef half8_t __attribute__((aligned(2))) half8_any_t;
template <int T, int NP>
struct Held {
    int lo, hi, edge;                          // whole pieces lo .. hi - 1; the element, or -1
    half8_t x[NP];
    half_t e;
    __device__ __forceinline__ Held(const VocabRow &z) : lo(z.off > 0), hi(max((z.V + z.off) / 8, lo))
    {
        const int head = lo ? min(8 - z.off, z.V) : 0, tail = max(8 * hi - z.off, head), j = (int)threadIdx.x < head ? (int)threadIdx.x : tail + (int)threadIdx.x - head;
        edge = threadIdx.x < 16 && j < z.V ? j : -1;
    }
    __device__ __forceinline__ bool has(int i) const { return lo + (int)threadIdx.x + i * T < hi; }
    __device__ __forceinline__ int piece(int i) const { return min(lo + (int)threadIdx.x + i * T, hi - 1); }
    __device__ __forceinline__ void load(const VocabRow &z, const VocabRow &of)        // (what it does not have is some other of the row)
    {
        e = z.row[max(edge, 0)];
        if (hi > lo)
#pragma unroll
            for (int i = 0; i < NP; i++) x[i] = *reinterpret_cast<const half8_any_t *>(z.row + of.first(piece(i)));
    }
};

// what is written where a gradient is, or is added to, `old`
__device__ __forceinline__ half_t combined(float d, int acc, half_t old) { return acc ? f2h(h2f(old) + rnd16(d)) : f2h(d); }

}  // namespace cacti
