// Pages of a cache handed out, shared, copied and packed, with all numbers on the device.  refs [P] counts who holds a page, a row of
// the table has a sequence's pages in order and -1 behind them.
//
//   fork     sequence b goes on as sequence parent[b]: its row becomes that one's, up to the pages that its positions take
//   fit      each sequence gets what its positions need: pages behind them go back, missing ones are the lowest free ones, in the
//            order of sequences and positions, and a page that is going to be written on by others too is copied first; one that there is
//            no page for stays with who holds it and is not written on, its entry -2 - page
//   compact  the held pages to the lowest places
//   copy     the pages that the other two say, of all layers' caches in one launch
//
// Fork is a launch over rows, whose counts are sums of whole numbers, in any order the same.  Fit and the scan of compact are one
// workgroup: what is free depends on everything that is given back, and a barrier costs less there than a launch (a batch's table and
// counts are some ten kilobytes).  Copying is bound by memory.
//
// On the device: fork 3 us for 8 as for 128 sequences, a launch's own time; fit 7.3 us for 8 sequences, 10.0 for 128, some six barriers with
// a look at memory between each two; copies of 8 to 128 pages 4.4 to 6.9; packing 6.6 + 4.6 us and its 492 MB of copies 95, 5.2 TB/s.
#include "common.h"

using namespace cacti;

namespace {

// Counts that one workgroup alone changes: past its first cache, no further
__device__ __forceinline__ int load_now(const int *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ __forceinline__ void store_now(int *p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ __forceinline__ void less_one(int *p) { __hip_atomic_fetch_add(p, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ __forceinline__ void one_more(int *p) { __hip_atomic_fetch_add(p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ __forceinline__ void no_more_than(int *p, int v) { __hip_atomic_fetch_min(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
// A barrier behind which the workgroup's counts in memory are what it made them: they are written and read past the first cache, in
// an order that the barrier alone does not promise.
__device__ __forceinline__ void settled()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0x0f70);        // vmcnt(0)
    __syncthreads();
}
__device__ __forceinline__ void name(int *status, int b)
{
    if (status) atomicMax(status, b + 1);
}
// The page that an entry holds, or an entry that holds none as it is
__device__ __forceinline__ int page_of(int x, int P) { return x < -1 && -2 - x < P ? -2 - x : x; }
__device__ __forceinline__ bool fits(int len, int W, int page) { return len >= 0 && len <= W * page; }

// ---------------------------------------------------------------- fork
struct ForkArgs {
    int P, B, W, page;
    int64_t ldt, ldn;
    int *refs;
    const int *table, *lens, *parent;
    int *new_table, *new_lens, *status;
};

// A workgroup to a sequence
__global__ void __launch_bounds__(256) fork_kernel(ForkArgs a)
{
    const int b = blockIdx.x;
    int p = a.parent[b], need = 0, len = 0;
    bool stays = p < -1 || p >= a.B;
    if (!stays && p >= 0) {
        len = a.lens[p];
        stays = !fits(len, a.W, a.page);
        need = (len + a.page - 1) / a.page;
    }
    if (stays) {                               // what cannot be: left as it is
        if (threadIdx.x == 0) name(a.status, b);
        p = b;
        len = a.lens[b];
        need = a.W;
    }
    const int *was = a.table + b * a.ldt, *from = a.table + max(p, 0) * a.ldt;
    int *to = a.new_table + b * a.ldn;
    for (int j = threadIdx.x; j < a.W; j += 256) {
        const int x = page_of(was[j], a.P), raw = j < need ? from[j] : -1, y = page_of(raw, a.P);
        to[j] = stays ? raw : y;
        if (x == y) continue;
        if (x >= 0 && x < a.P) atomicSub(a.refs + x, 1);
        if (y >= 0 && y < a.P) atomicAdd(a.refs + y, 1);
    }
    if (threadIdx.x == 0) a.new_lens[b] = len;
}

// ---------------------------------------------------------------- fit
struct FitArgs {
    int P, B, W, page;
    int64_t ldt;
    int *refs, *table;
    const int *first, *lens;
    int *src, *dst, *slots;
    int *asked, *free;                         // workspace: [B] pages that each sequence asks for, [P] free ones in order
    int *status;
};

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// the sum over the threads before this one, and of all
__device__ __forceinline__ int scan(int v, int *total, int *red)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(s, o);
        if (lane >= o) s += x;
    }
    __syncthreads();
    if (lane == 63) red[wave] = s;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        const int x = red[w];
        before += w < wave ? x : 0;
        sum += x;
    }
    *total = sum;
    return before + s - v;
}

// found(page, the wave's lanes whose page is one, how many are before the wave's) for the D 1024 pages from p0 on, D to a thread, whose counts
// are on their way together; how many there are
constexpr int kDeep = 16;
__device__ __forceinline__ bool mine(uint64_t mask) { return __builtin_amdgcn_inverse_ballot_w64(mask); }
__device__ __forceinline__ int before_mine(uint64_t mask) { return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0)); }
template <int D, class Is, class Found>
__device__ __forceinline__ int look(const int *refs, int p0, int hi, int all, int *counts, Is is, Found found)
{
    constexpr int kOwn = (kWaves * D + 63) / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), p = p0 + (int)threadIdx.x;
    int held[D], own = 0;
    uint64_t mask[D];
#pragma unroll
    for (int k = 0; k < D; k++) held[k] = load_now(refs + min(p + k * kThreads, hi - 1));
#pragma unroll
    for (int k = 0; k < D; k++) {
        mask[k] = __ballot(p + k * kThreads < hi && is(held[k]));
        own = lane == k ? __popcll(mask[k]) : own;
    }
    if (lane < D) counts[kWaves * lane + wave] = own;
    __syncthreads();
    // counts of the waves, then those 1024 pages further: a lane has kOwn of them
    int c[kOwn], s = 0;
#pragma unroll
    for (int i = 0; i < kOwn; i++) c[i] = kOwn * lane + i < kWaves * D ? counts[kOwn * lane + i] : 0, s += c[i];
    int before = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(before, o);
        if (lane >= o) before += x;
    }
    const int total = __builtin_amdgcn_readlane(before, 63);
    before += all - s;
#pragma unroll
    for (int i = 0; i < kOwn - 1; i++) before += i < wave % kOwn ? c[i] : 0;
#pragma unroll
    for (int k = 0; k < D; k++) found(p + k * kThreads, mask[k], __builtin_amdgcn_readlane(before, (kWaves * k + wave) / kOwn));
    __syncthreads();
    return total;
}
// .. from lo on until `most` are found or to the end, up to 16384 pages at a time, in two barriers and a round trip to memory.  (Fit with 30000
// pages to look through takes 4 us longer, with 100000 16; by 4096 at a time 10 and 35.  Packing 100000 takes 60 us, by 1024 120.)
template <class Is, class Found>
__device__ __forceinline__ int search(const int *refs, int lo, int hi, int most, int *counts, Is is, Found found)
{
    int all = 0;
    for (int64_t p = lo; p < hi && all < most;) {
        const int64_t left = hi - p;
        const int deep = left <= kThreads ? 1 : left <= 4 * kThreads ? 4 : kDeep;
        if (deep == 1) all += look<1>(refs, (int)p, hi, all, counts, is, found);
        else if (deep == 4) all += look<4>(refs, (int)p, hi, all, counts, is, found);
        else all += look<kDeep>(refs, (int)p, hi, all, counts, is, found);
        p += deep * kThreads;
    }
    return all;
}

// A sequence's entries that it lets go of, those from begin on, of which those below need are wanted again; part: slots of the first
// one that are to be kept.  What does not fit together lets go of nothing.
struct Span {
    int begin, need, part;
};
__device__ __forceinline__ Span span(const FitArgs &a, int b, bool *ok)
{
    const int f = a.first[b], l = a.lens[b];
    *ok = fits(l, a.W, a.page) && f >= 0 && f <= l;
    if (!*ok) return {a.W, 0, 0};
    const int need = (int)((unsigned)(l + a.page - 1) / (unsigned)a.page), whole = (int)((unsigned)f / (unsigned)a.page);
    return {l > f ? whole : need, need, l > f ? f - whole * a.page : 0};
}

constexpr int kHeld = 2048;                    // sequences whose spans are in LDS
constexpr int kLanes = 8;                      // that look at the entries of a sequence which it lets go of and wants again: most have 1 to 3
// f(sequence, its span, entry of the lane's own or one behind the last, whether it is the first time)
template <class F>
__device__ __forceinline__ void each(const FitArgs &a, const Span *held, F f)
{
    for (int b = threadIdx.x / kLanes; b < a.B; b += kThreads / kLanes) {
        bool ok;
        const Span s = b < kHeld ? held[b] : span(a, b, &ok);
        for (int j = s.begin; j < s.need; j += kLanes) f(b, s, j + (int)threadIdx.x % kLanes, j == s.begin);
    }
}
// the lanes of a sequence of which something holds
__device__ __forceinline__ int lanes_with(bool x) { return (int)(__ballot(x) >> (threadIdx.x & 63 & ~(kLanes - 1))) & ((1 << kLanes) - 1); }

__global__ void __launch_bounds__(kThreads) fit_kernel(FitArgs a)
{
    __shared__ int red[kWaves], counts[kWaves * kDeep];
    __shared__ Span held[kHeld];
    auto entry = [&](int b, int j) __attribute__((always_inline)) { return a.table + b * a.ldt + j; };
    auto page = [&](int x) __attribute__((always_inline)) { return x >= 0 && x < a.P; };
    auto held_by = [&](const int *entry) __attribute__((always_inline)) { return page_of(*entry, a.P); };
    for (int b = threadIdx.x; b < a.B; b += kThreads) {
        bool ok;
        const Span s = span(a, b, &ok);
        if (b < kHeld) held[b] = s;
        if (!ok) name(a.status, b);
        a.src[b] = a.dst[b] = -1;
        a.slots[b] = a.asked[b] = 0;
    }
    __syncthreads();
    // what is not needed goes back; some entries under way together
    {
        constexpr int kAhead = 4;
        int b = (int)threadIdx.x / a.W, j = (int)threadIdx.x - b * a.W;
        const int db = kThreads / a.W, dj = kThreads - db * a.W;
        while (b < a.B) {
            int x[kAhead], *at[kAhead];
            bool gone[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                bool ok;
                const int own = min(b, a.B - 1);
                const Span s = own < kHeld ? held[own] : span(a, own, &ok);
                gone[i] = b < a.B && j >= s.begin && j >= s.need;
                at[i] = entry(own, j);
                x[i] = *at[i];
                b += db, j += dj;
                if (j >= a.W) b++, j -= a.W;
            }
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                if (!gone[i]) continue;
                const int own = page_of(x[i], a.P);
                if (page(own)) less_one(a.refs + own);
                if (x[i] != -1) *at[i] = -1;
            }
        }
    }
    // what is written on is let go of
    each(a, held, [&](int b, const Span &s, int j, bool) __attribute__((always_inline)) {
        const int x = j < s.need ? held_by(entry(b, j)) : -1;
        if (page(x)) less_one(a.refs + x);
    });
    settled();
    // a page that no one keeps goes to the first of those who want it again: b - B, below all counts
    each(a, held, [&](int b, const Span &s, int j, bool) __attribute__((always_inline)) {
        const int x = j < s.need ? held_by(entry(b, j)) : -1;
        if (page(x) && load_now(a.refs + x) <= 0) no_more_than(a.refs + x, b - a.B);
    });
    settled();
    // who has none of its own asks for one
    each(a, held, [&](int b, const Span &s, int j, bool first) __attribute__((always_inline)) {
        const int raw = j < s.need ? *entry(b, j) : -1, x = page_of(raw, a.P);
        const bool asks = j < s.need && !(page(x) && load_now(a.refs + x) == b - a.B);
        if (asks && s.part && j == s.begin && page(x)) a.src[b] = x;
        if (asks) *entry(b, j) = -1;
        else if (x != raw) *entry(b, j) = x;
        const int n = __popc(lanes_with(asks));
        if (threadIdx.x % kLanes == 0) a.asked[b] = (first ? 0 : a.asked[b]) + n;
    });
    settled();
    // how many are asked for before each sequence
    int all = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
        const int b = b0 + (int)threadIdx.x;
        int total;
        const int before = scan(b < a.B ? a.asked[b] : 0, &total, red);
        if (b < a.B) a.asked[b] = all + before;
        all += total;
    }
    // the lowest free pages, as many as are asked for
    const int found = search(a.refs, 0, a.P, all, counts, [](int r) { return r == 0; }, [&](int p, uint64_t are, int at) __attribute__((always_inline)) {
        if (mine(are)) a.free[at + before_mine(are)] = p;
    });
    settled();
    // .. handed out; what is kept counts one
    int at = 0;
    each(a, held, [&](int b, const Span &s, int j, bool first) __attribute__((always_inline)) {
        if (first) at = a.asked[b];
        int x = j < s.need ? *entry(b, j) : -2;
        const bool asks = x == -1;
        const int mask = lanes_with(asks), k = at + __popc(mask & ((1 << threadIdx.x % kLanes) - 1));
        at += __popc(mask);
        if (asks && k < found) *entry(b, j) = x = a.free[k];
        if (x >= 0) store_now(a.refs + x, 1);
        if (!asks) return;
        const bool copied = s.part && j == s.begin && a.src[b] >= 0;
        if (x < 0) name(a.status, b);
        if (copied && x >= 0) a.dst[b] = x, a.slots[b] = s.part;
    });
    if (found >= all) return;
    // pages ran out: what was to be copied and cannot be stays with its sequence
    settled();
    for (int b = threadIdx.x; b < a.B; b += kThreads) {
        if (a.src[b] < 0 || a.dst[b] >= 0) continue;
        bool ok;
        one_more(a.refs + a.src[b]);
        *entry(b, span(a, b, &ok).begin) = -2 - a.src[b];
        a.src[b] = -1;
    }
    settled();
    // .. and who would have kept such a page for itself does not write on it either
    each(a, held, [&](int b, const Span &s, int j, bool) __attribute__((always_inline)) {
        const int x = j < s.need ? *entry(b, j) : -1;
        if (x < 0 || load_now(a.refs + x) <= 1) return;
        name(a.status, b);
        const bool part = s.part && j == s.begin;
        *entry(b, j) = part ? -2 - x : -1;
        if (!part) less_one(a.refs + x);
    });
}

// ---------------------------------------------------------------- compact
struct CompactArgs {
    int P, B, W;
    int64_t ldt;
    int *refs, *table, *src, *dst, *used;
    int *to;                                   // workspace [P]: where a page goes that moves
};

__global__ void __launch_bounds__(kThreads) compact_kernel(CompactArgs a)
{
    __shared__ int counts[kWaves * kDeep];
    auto is_held = [](int r) { return r > 0; };
    const int half = a.P / 2;
    for (int i = threadIdx.x; i < half; i += kThreads) a.src[i] = a.dst[i] = -1;
    const int used = search(a.refs, 0, a.P, a.P, counts, is_held, [](int, uint64_t, int) {});
    if (threadIdx.x == 0) *a.used = used;
    // free places below `used` and held pages from there on: as many of the one as of the other
    search(a.refs, 0, used, used, counts, [](int r) { return r <= 0; }, [&](int p, uint64_t are, int at) __attribute__((always_inline)) {
        if (mine(are)) a.dst[at + before_mine(are)] = p;
    });
    const int moves = search(a.refs, used, a.P, a.P, counts, is_held, [&](int p, uint64_t are, int at) __attribute__((always_inline)) {
        if (mine(are)) a.src[at + before_mine(are)] = p;
        else if (p < a.P) a.to[p] = p;
    });
    __syncthreads();
    for (int i = threadIdx.x; i < moves; i += kThreads) {
        const int s = a.src[i], d = a.dst[i];
        a.refs[d] = a.refs[s];
        a.refs[s] = 0;
        a.to[s] = d;
    }
}

__global__ void __launch_bounds__(256) renumber_kernel(CompactArgs a)
{
    const int used = *a.used;
    int *row = a.table + blockIdx.x * a.ldt;
    for (int j = threadIdx.x; j < a.W; j += 256) {
        const int x = row[j], p = page_of(x, a.P);
        if (p >= used && p < a.P) row[j] = x < 0 ? -2 - a.to[p] : a.to[p];
    }
}

// ---------------------------------------------------------------- copy
constexpr int kLayers = 32;
struct CopyArgs {
    char *k[kLayers], *v[kLayers];
    float *ks[kLayers], *vs[kLayers];
    const int *src, *dst, *slots;
    int64_t P;
    unsigned items;
    int parts, layers, heads, page, slot_bytes;        // (of a position of a head)
};

// An item: four heads of the keys or the values of a page of a layer, a wave to each
__global__ void __launch_bounds__(256) copy_kernel(CopyArgs a)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (unsigned i = blockIdx.x; i < a.items; i += gridDim.x) {
        const unsigned part = i % a.parts, of = i / a.parts % (2 * a.layers), which = i / a.parts / (2 * a.layers), layer = of >> 1;
        const int64_t s = a.src[which], d = a.dst[which];
        if (s < 0 || d < 0 || s >= a.P || d >= a.P || s == d) continue;
        const int slots = a.slots ? min(max(a.slots[which], 0), a.page) : a.page, h = 4 * (int)part + wave;
        if (h >= a.heads || slots == 0) continue;
        const int64_t head = (int64_t)a.page * a.slot_bytes;
        char *pages = of & 1 ? a.v[layer] : a.k[layer];
        const uint4 *from = reinterpret_cast<const uint4 *>(pages + (s * a.heads + h) * head);
        uint4 *to = reinterpret_cast<uint4 *>(pages + (d * a.heads + h) * head);
        const int pieces = slots * a.slot_bytes / 16;
        int e = lane;
        for (; e + 192 < pieces; e += 256) {   // 4 KB under way
            const uint4 x0 = from[e], x1 = from[e + 64], x2 = from[e + 128], x3 = from[e + 192];
            to[e] = x0, to[e + 64] = x1, to[e + 128] = x2, to[e + 192] = x3;
        }
        for (; e < pieces; e += 64) to[e] = from[e];
        float *scales = of & 1 ? a.vs[layer] : a.ks[layer];
        if (scales && lane == 0) scales[d * a.heads + h] = scales[s * a.heads + h];
    }
}

int check(const char *who, int64_t P, int64_t B, int64_t W, int64_t page, const void *refs, const void *table, int64_t ldt, const void *status)
{
    CACTI_REQUIRE(P > 0 && B > 0 && W > 0 && page > 0, CACTI_E_INVALID, "%s: empty shape", who);
    CACTI_REQUIRE(refs && table, CACTI_E_INVALID, "%s: null pointer", who);
    CACTI_REQUIRE(P <= (1 << 28) && B <= (1 << 20) && W <= (1 << 30) / page && B * W <= INT32_MAX && ldt >= W, CACTI_E_NOTIMPL,
                  "%s: too many pages or sequences, or a table pitch below its width", who);
    CACTI_REQUIRE(aligned(refs, 4) && aligned(table, 4) && aligned(status, 4), CACTI_E_INVALID, "%s: misaligned operand", who);
    return 0;
}

}  // namespace

CACTI_API int cacti_hip_paged_fork(int64_t P, int64_t B, int64_t W, int64_t page, void *refs, const void *table, int64_t ldt, const void *lens,
                                   const void *parent, void *new_table, int64_t ldn, void *new_lens, void *status, void *stream)
{
    const int rc = check("paged_fork", P, B, W, page, refs, table, ldt, status);
    if (rc) return rc;
    CACTI_REQUIRE(lens && parent && new_table && new_lens, CACTI_E_INVALID, "paged_fork: null pointer");
    CACTI_REQUIRE(aligned(lens, 4) && aligned(parent, 4) && aligned(new_table, 4) && aligned(new_lens, 4), CACTI_E_INVALID, "paged_fork: misaligned operand");
    CACTI_REQUIRE(ldn >= W, CACTI_E_INVALID, "paged_fork: a table pitch below its width");
    auto share = [](const void *a, int64_t na, const void *b, int64_t nb) {      // na numbers at a, nb at b
        const char *p = (const char *)a, *q = (const char *)b;
        return p < q + 4 * nb && q < p + 4 * na;
    };
    const int64_t size = (B - 1) * ldn + W;
    CACTI_REQUIRE(!share(new_table, size, table, (B - 1) * ldt + W), CACTI_E_INVALID, "paged_fork: the new table shares memory with the old one");
    CACTI_REQUIRE(!share(new_lens, B, lens, B), CACTI_E_INVALID, "paged_fork: the new lengths share memory with the old ones");
    // (a sequence's row and length are written while others' are read)
    CACTI_REQUIRE(!share(new_table, size, lens, B) && !share(new_table, size, parent, B) && !share(new_table, size, refs, P) && !share(new_table, size, new_lens, B) &&
                      !share(new_lens, B, parent, B) && !share(new_lens, B, refs, P) && !share(new_lens, B, table, (B - 1) * ldt + W),
                  CACTI_E_INVALID, "paged_fork: the new table or the new lengths share memory with another operand");
    const ForkArgs a = {(int)P, (int)B, (int)W, (int)page, ldt, ldn, (int *)refs, (const int *)table, (const int *)lens, (const int *)parent,
                        (int *)new_table, (int *)new_lens, (int *)status};
    hipLaunchKernelGGL(fork_kernel, dim3((unsigned)B), dim3(256), 0, (hipStream_t)stream, a);
    return launch_status("paged_fork");
}

CACTI_API size_t cacti_hip_paged_fit_workspace(int64_t P, int64_t B) { return P > 0 && B > 0 ? (size_t)(P + B) * 4 : 0; }

CACTI_API int cacti_hip_paged_fit(int64_t P, int64_t B, int64_t W, int64_t page, void *refs, void *table, int64_t ldt, const void *first,
                                  const void *lens, void *src, void *dst, void *slots, void *workspace, size_t workspace_bytes, void *status,
                                  void *stream)
{
    const int rc = check("paged_fit", P, B, W, page, refs, table, ldt, status);
    if (rc) return rc;
    CACTI_REQUIRE(first && lens && src && dst && slots && workspace, CACTI_E_INVALID, "paged_fit: null pointer");
    CACTI_REQUIRE(aligned(first, 4) && aligned(lens, 4) && aligned(src, 4) && aligned(dst, 4) && aligned(slots, 4) && aligned(workspace, 4), CACTI_E_INVALID,
                  "paged_fit: misaligned operand");
    CACTI_REQUIRE(workspace_bytes >= cacti_hip_paged_fit_workspace(P, B), CACTI_E_INVALID, "paged_fit: workspace of %zu bytes, %zu needed", workspace_bytes,
                  cacti_hip_paged_fit_workspace(P, B));
    const FitArgs a = {(int)P, (int)B, (int)W, (int)page, ldt, (int *)refs, (int *)table, (const int *)first, (const int *)lens, (int *)src, (int *)dst,
                       (int *)slots, (int *)workspace, (int *)workspace + B, (int *)status};
    hipLaunchKernelGGL(fit_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, a);
    return launch_status("paged_fit");
}

CACTI_API size_t cacti_hip_paged_compact_workspace(int64_t P) { return P > 0 ? (size_t)P * 4 : 0; }

CACTI_API int cacti_hip_paged_compact(int64_t P, int64_t B, int64_t W, void *refs, void *table, int64_t ldt, void *src, void *dst, void *used,
                                      void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = check("paged_compact", P, B, W, 1, refs, table, ldt, nullptr);
    if (rc) return rc;
    CACTI_REQUIRE(((src && dst) || P < 2) && used && workspace, CACTI_E_INVALID, "paged_compact: null pointer");
    CACTI_REQUIRE(aligned(src, 4) && aligned(dst, 4) && aligned(used, 4) && aligned(workspace, 4), CACTI_E_INVALID, "paged_compact: misaligned operand");
    CACTI_REQUIRE(workspace_bytes >= cacti_hip_paged_compact_workspace(P), CACTI_E_INVALID, "paged_compact: workspace of %zu bytes, %zu needed",
                  workspace_bytes, cacti_hip_paged_compact_workspace(P));
    const CompactArgs a = {(int)P, (int)B, (int)W, ldt, (int *)refs, (int *)table, (int *)src, (int *)dst, (int *)used, (int *)workspace};
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, a);
    hipLaunchKernelGGL(renumber_kernel, dim3((unsigned)B), dim3(256), 0, (hipStream_t)stream, a);
    return launch_status("paged_compact");
}

CACTI_API int cacti_hip_paged_copy(int64_t layers, void *const *k_pages, void *const *v_pages, void *const *k_scale, void *const *v_scale, int bits,
                                   int64_t P, int64_t Hkv, int64_t page, int64_t Dh, int64_t n, const void *src, const void *dst, const void *slots,
                                   void *stream)
{
    CACTI_REQUIRE(layers >= 0 && P > 0 && Hkv > 0 && page > 0 && Dh > 0 && n >= 0, CACTI_E_INVALID, "paged_copy: empty shape");
    CACTI_REQUIRE(bits == 8 || bits == 16, CACTI_E_INVALID, "paged_copy: pages of 8 or 16 bits");
    CACTI_REQUIRE(Dh <= 4096 && page <= 4096 && Hkv <= 4096 && P <= (1 << 28) && n <= (1 << 28) && layers <= (1 << 16), CACTI_E_NOTIMPL,
                  "paged_copy: pages too large or too many");
    CACTI_REQUIRE(Hkv * page * ((Dh + 15) / 16 * 16) * (bits / 8) <= (1 << 30), CACTI_E_NOTIMPL, "paged_copy: pages too large or too many");
    if (layers == 0 || n == 0) return 0;
    CACTI_REQUIRE(k_pages && v_pages && src && dst && (bits == 16 || (k_scale && v_scale)), CACTI_E_INVALID, "paged_copy: null pointer");
    CACTI_REQUIRE(aligned(src, 4) && aligned(dst, 4) && aligned(slots, 4), CACTI_E_INVALID, "paged_copy: misaligned operand");
    for (int64_t l = 0; l < layers; l++) {
        CACTI_REQUIRE(k_pages[l] && v_pages[l] && aligned(k_pages[l], 16) && aligned(v_pages[l], 16), CACTI_E_INVALID,
                      "paged_copy: pages null or not 16-byte aligned");
        CACTI_REQUIRE(bits == 16 || (k_scale[l] && v_scale[l] && aligned(k_scale[l], 4) && aligned(v_scale[l], 4)), CACTI_E_INVALID,
                      "paged_copy: pages of 8 bits have scales");
    }
    for (int64_t l0 = 0; l0 < layers; l0 += kLayers) {
        CopyArgs a{};
        a.layers = (int)(layers - l0 < kLayers ? layers - l0 : kLayers);
        for (int l = 0; l < a.layers; l++) {
            a.k[l] = (char *)k_pages[l0 + l], a.v[l] = (char *)v_pages[l0 + l];
            if (bits == 8) a.ks[l] = (float *)k_scale[l0 + l], a.vs[l] = (float *)v_scale[l0 + l];
        }
        a.src = (const int *)src, a.dst = (const int *)dst, a.slots = (const int *)slots;
        a.heads = (int)Hkv, a.page = (int)page, a.slot_bytes = (int)((Dh + 15) / 16 * 16 * bits / 8);
        const int64_t parts = (Hkv + 3) / 4, items = n * 2 * a.layers * parts;
        CACTI_REQUIRE(items <= INT32_MAX, CACTI_E_NOTIMPL, "paged_copy: too many pages");
        a.P = P, a.parts = (int)parts, a.items = (unsigned)items;
        const int64_t blocks = a.items < 4096 ? a.items : 4096;
        hipLaunchKernelGGL(copy_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
    }
    return launch_status("paged_copy");
}
