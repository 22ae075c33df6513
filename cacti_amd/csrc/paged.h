// A ragged batch of sequences over a paged key / value cache, as the kernels that write (paged_append.hip) and read it
// (paged_attention.hip) see it.
//
// Rows starts[b] .. starts[b + 1] - 1 of the batch are the new tokens of sequence b, lens[b] its positions with them: its row i
// is at position lens[b] - n + i.  Position p lies in slot p % page of page table[b][p / page].  These numbers are device
// memory, unknown to the host that launches: a sequence whose numbers do not fit together is left out and named in `status`.
#pragma once
#include "common.h"

namespace cacti {

struct PagedBatch {
    int T, B;                       // rows there are, sequences
    int page, W;                    // positions of a page; pages of a row of the table
    int64_t ldt;                    // row pitch of the table
    int P;                          // pages of the cache
    const int *starts, *lens, *table;
    int *status;                    // null, or 1 + the sequence that was left out
};

// pages of a head in bytes: rows of a position padded to 16 elements
__host__ __device__ inline int padded_dim(int Dh) { return (Dh + 15) & ~15; }

__device__ __forceinline__ void report(const PagedBatch &pb, int b)
{
    if (pb.status) atomicMax(pb.status, b + 1);
}

// A sequence's rows: s0 .. s0 + n - 1 at positions first .. first + n - 1.  ok: these are rows and positions that there are.
struct Sequence {
    int s0, n, first;
    bool ok;
};
__device__ __forceinline__ Sequence sequence(const PagedBatch &pb, int b, int64_t limit, int max_new)
{
    Sequence q;
    const int s1 = pb.starts[b + 1], len = pb.lens[b];
    q.s0 = pb.starts[b];
    q.n = (int)((unsigned)s1 - (unsigned)q.s0);            // (any numbers: what of this does not fit into 32 bits is not ok)
    q.first = (int)((unsigned)len - (unsigned)q.n);
    q.ok = q.s0 >= 0 && s1 >= q.s0 && s1 <= pb.T && q.n <= max_new && len >= q.n && len <= limit;
    return q;
}

// A lane's sequence of 64 from b0 on, and a lane's to all of the wave
__device__ __forceinline__ Sequence lane_sequence(const PagedBatch &pb, int b0, int64_t limit, int max_new)
{
    const int b = b0 + (threadIdx.x & 63);
    Sequence s = sequence(pb, min(b, pb.B - 1), limit, max_new);
    if (b >= pb.B) s.n = 0, s.ok = false;
    return s;
}
__device__ __forceinline__ Sequence of_lane(const Sequence &s, int lane)
{
    return {__builtin_amdgcn_readlane(s.s0, lane), __builtin_amdgcn_readlane(s.n, lane), __builtin_amdgcn_readlane(s.first, lane),
            __builtin_amdgcn_readlane((int)s.ok, lane) != 0};
}

// How many of f(1) .. f(B) are <= x, for an f that does not fall: the sequence that unit x of them belongs to.  Every lane
// of a wave that calls looks at some (one round trip to memory for up to 64 sequences) and all get the answer.
template <class F>
__device__ __forceinline__ int count_below(int B, int64_t x, F f)
{
    const int lane = threadIdx.x & 63;
    int c = 0;
    for (int i0 = 1; i0 <= B; i0 += 64) {
        const int i = i0 + lane;
        c += __popcll(__ballot(i <= B && f(i) <= x));
    }
    return c;
}

// Units of the sequences of a launch (pages they touch, tiles of their rows) are numbered so that the host need not know the
// lengths.  even > 0: `even` numbers for each sequence.  Otherwise a sequence of rows s0 .. s1 - 1 has those from
// s0 / per times + more b on: at least (s1 - s0) / per times + more of them, which has to be enough for its n rows.
struct Units {
    int even, per, times, more;
    int64_t count;
    __device__ __forceinline__ int64_t begin(int b, int s0) const { return even ? (int64_t)b * even : (int64_t)(max(s0, 0) / per) * times + (int64_t)more * b; }
    __device__ __forceinline__ int64_t first(const PagedBatch &pb, int i) const { return begin(i, pb.starts[i]); }
    // (sequence, unit of it) of number x; sequence B: none
    __device__ __forceinline__ int find(const PagedBatch &pb, int64_t x, int *unit) const
    {
        if (even) {
            const int b = (int)(x / even);
            *unit = (int)(x - (int64_t)b * even);
            return b;
        }
        const int b = count_below(pb.B, x, [&](int i) { return first(pb, i); });
        *unit = b < pb.B ? (int)(x - first(pb, b)) : 0;
        return b;
    }
};
// units of a launch over T rows: `most` for a sequence of max_new rows
inline Units make_units(int64_t T, int64_t B, int64_t per, int64_t times, int more, int64_t most)
{
    const int64_t searched = T / per * times + (int64_t)more * B;
    if (most * B <= searched) return {(int)most, (int)per, (int)times, more, most * B};
    return {0, (int)per, (int)times, more, searched};
}

// What is the same of the calls' checks; sets pb
int paged_batch(const char *who, int64_t T, int64_t B, int64_t H, int64_t Hkv, int64_t Dh, int64_t max_new, const void *table,
                int64_t ldt, int64_t W, const void *starts, const void *lens, void *status, const void *k_pages, const void *v_pages,
                const void *k_scale, const void *v_scale, int bits, int64_t P, int64_t page, PagedBatch *pb);

}  // namespace cacti
