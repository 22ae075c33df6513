// Causal attention of the new rows of a ragged batch over a paged cache, in e4m3 with a scale per page and head or in f16:
//   o = sum_j softmax_j(alpha q . k_j) v_j     over the positions j up to the row's own
//
// One pass over the keys with a running m, the maximum of a row's scores so far (or, prompts in 16 bits, up to kSlack less).  The codes
// meet the queries as they are (e4m3 to f16 is exact) and a page's scales join the scores: with t_j = alpha ks q . k_j log2 e + log2 vs,
//   w_j = 2^(15 + t_j - m),  o = sum w_j code(v_j) / sum w_j / vs
// so that the weight that meets a code already holds its page's scale, and no w exceeds f16 whatever the scales are.  The largest w is
// 2^15, at the upper end of f16, to leave those of a row's other pages their bits down to 2^-29 of it: with 1 for the largest, one large
// value in a page, 2^18 above the others, cost those 4 bits of their 11.
// Scores, maxima, sums and o are fp32; w is rounded to f16 for the matrix instruction (2^-11 relative, each on its own, which
// is what the rounding of the output adds once more).  The sum is that of w as it was, since a page of small values may have
// weights that are nothing in f16 and most of the probability; the largest w is a power of two, and exact.  With kSlack it need not be,
// but there are no scales then: the sum is that of the rounded w, and what a large one is off by is off in both.
//
// A wave takes 16 NR rows (tokens of a sequence by the query heads that share a key head) of a key head at a time, by itself, 32
// positions at a time.  The products are formed transposed, S^T = K Q^T and O^T = V^T W^T with v_mfma_f32_16x16x32_f16: a lane
// then holds the scores of one row, at keys that are exactly those its part of the second product's operand wants, so that w
// never leaves the lane.  Keys come from memory in the order the instruction takes them (16 columns of a key to a lane); V, whose
// operand is a column of eight keys, is read as rows of 8 columns and turned with byte permutes.  LDS has the pages' numbers and
// no operand, and nobody waits on the way; the keys after these are requested once these have been multiplied, the values likewise,
// into the same registers.  48 sequences of 120 to 8192 positions, 32 heads of 100 in 8 bits, which memory bounds: 129 us, 24 of 100 to
// 6000 with up to 6 rows of 32 / 8 heads of 128, vector operations as much as memory: 27.5 us; one of 1540, latency: 12.3 us; the first
// two in 16 bits, which memory bounds: 236 and 41.7 us.
//
// Work: the lengths are on the device and as different as they come, so every workgroup of a launch that just fills the device
// forms their sum in steps of 32 positions and takes an equal, contiguous share of it, across rows, heads and sequences, each of
// its waves a quarter.  What its waves have of a tile of rows they put together in LDS; a tile that ends up in more than one
// share leaves partial sums, which a second launch puts together.
#include "operands.h"
#include "paged.h"
#include "paged_shares.h"

using namespace cacti;

namespace {

using namespace cacti::shares;

constexpr int kThreads = 64 * kWaves;

struct AttnArgs {
    PagedBatch pb;
    int H, Hkv, G, Dh, Dp, max_new, groups;
    unsigned page_magic;                       // x / page = x * page_magic >> 22 for x below kEntries pages
    float alpha;                               // |alpha|; its sign goes to the queries
    unsigned sign;                             // 0x80008000 where it is negative
    const half_t *q;
    int64_t ldq;
    const void *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    half_t *out;
    int64_t ldo;
    float *part, *stats;                       // [2 groups][16 NR][Dh], [2 groups][16 NR][2]; a group: a workgroup
    int few;                                   // sequences with more rows than that (by the query heads of a key head) are prompts
    int big_groups;                            // ... for which a group is a workgroup; 0: there are none
    float *big_part, *big_stats;               // [2 big_groups][kPrompt][Dh], ...[2]
};

// What is the same in all lanes, in scalar registers
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// The lane's number, of which the compiler does not know that it is the same every time: what is formed from it for one tile of
// rows (some hundred addresses) is formed there and not held in registers, or out of them, over all tiles of a share.
__device__ __forceinline__ int lane_here()
{
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// A sequence's share of the work, as one of few rows and as a prompt
__device__ __forceinline__ Share share_of(const AttnArgs &a, int tile, const Sequence &s)
{
    return Share(tile, s.n * a.G, s.first + s.n, a.Hkv, s.ok && s.n > 0 && s.n * a.G <= a.few);
}
__device__ __forceinline__ BigShare big_share_of(const AttnArgs &a, const Sequence &s) { return BigShare(a.G, s.n * a.G, s.first, s.ok && s.n * a.G > a.few); }
__device__ __forceinline__ Sequence lane_sequence(const AttnArgs &a, int b0)
{
    return lane_sequence(a.pb, b0, (int64_t)a.pb.W * a.pb.page, a.max_new);
}

// Work is counted in 32 bits; the host has seen to it that rows which each are of one sequence are not more.  (Where starts fall a row may
// be of many: nothing is done then.)
__device__ __forceinline__ bool too_much(double units) { return units > (double)INT32_MAX; }

// Workgroups go round the 8 XCDs: those of one XCD get neighbouring numbers (of n, a multiple of 8)
__device__ __forceinline__ unsigned xcd_order(unsigned i, unsigned n) { return (i & 7) * (n / 8) + i / 8; }

typedef unsigned u4_t __attribute__((ext_vector_type(4)));
typedef unsigned u2_t __attribute__((ext_vector_type(2)));

union Frag {
    half8_t h;
    unsigned u[4];
};

__device__ __forceinline__ unsigned cvt8(unsigned w, bool high)
{
    return high ? __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}

// 16 columns of a key: one piece of 16 codes, or two of 8 halves
template <class P>
struct KPiece;
template <>
struct KPiece<uint8_t> {
    u4_t w;
    __device__ __forceinline__ void load(const uint8_t *p) { w = *reinterpret_cast<const u4_t *>(p); }
};
template <>
struct KPiece<half_t> {
    half8_t w[2];
    __device__ __forceinline__ void load(const half_t *p)
    {
        w[0] = *reinterpret_cast<const half8_t *>(p);
        w[1] = *reinterpret_cast<const half8_t *>(p + 8);
    }
    __device__ __forceinline__ void zero() { w[0] = w[1] = half8_t{}; }
};

typedef int i8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The lane's part of a query: of each 64 columns those that it has of a key.
template <int ND>
struct QueryWords {
    u2_t w[4 * ND];                            // as loaded: word i at column 64 (i / 4) + 16 g + 4 (i % 4)
    __device__ __forceinline__ void load(const half_t *q, int Dh, int g)   // (Dh is a multiple of 4)
    {
#pragma unroll
        for (int i = 0; i < 4 * ND; i++) w[i] = *reinterpret_cast<const u2_t *>(q + min(64 * (i / 4) + 16 * g + 4 * (i & 3), Dh - 4));
    }
    __device__ __forceinline__ u2_t at(int i, int Dh, unsigned sign) const
    {
        return 64 * (i / 4) + 16 * (int)((threadIdx.x & 63) >> 4) + 4 * (i & 3) < Dh ? w[i] ^ sign : u2_t{0u, 0u};
    }
};
template <int ND, class P>
struct Query;
template <int ND>
struct Query<ND, half_t> {
    half8_t h[2 * ND];
    __device__ __forceinline__ float set(const QueryWords<ND> &q, int Dh, unsigned sign)  // returns what the products have to be multiplied by
    {
#pragma unroll
        for (int c = 0; c < 2 * ND; c++) {
            Frag x;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const u2_t w = q.at(2 * c + j, Dh, sign);
                x.u[2 * j] = w[0];
                x.u[2 * j + 1] = w[1];
            }
            h[c] = x.h;
        }
        return 1.f;
    }
    __device__ __forceinline__ float4_t times(const KPiece<half_t> (&k)[ND]) const
    {
        float4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2 * ND; c++) s = mfma(k[c / 2].w[c & 1], h[c], s);
        return s;
    }
};
// Against codes: three e4m3 terms, each the rounded rest of those before, of the query scaled by a power of two to have its
// largest element between 224 and 448.  They have 4 + 5 + 5 bits, and so all 11 of an element of at least 1/112 of the largest
// (below, they are off by 2^-10, 2^-18 of the largest); the codes need no conversion, which is 32 vector operations of 64
// columns by 32 keys, and the products of 8 bits have the matrix pipe to themselves.
template <int ND>
struct Query<ND, uint8_t> {
    int t[3][4 * ND];
    __device__ __forceinline__ float set(const QueryWords<ND> &q, int Dh, unsigned sign)
    {
        float x[16 * ND], mx = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * ND; i++) {
            const half4_t w = __builtin_bit_cast(half4_t, q.at(i, Dh, sign));
#pragma unroll
            for (int k = 0; k < 4; k++) {
                x[4 * i + k] = h2f(w[k]);
                mx = fmaxf(mx, fabsf(x[4 * i + k]));
            }
        }
        mx = with32(with16(mx, OpMax()), OpMax());
        int e = 0;
        if (mx > 0.f && mx < INFINITY) e = __builtin_amdgcn_frexp_expf(mx) - (__builtin_amdgcn_frexp_mantf(mx) > 0.875f ? 8 : 9);
#pragma unroll
        for (int i = 0; i < 4 * ND; i++) {
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = __builtin_amdgcn_ldexpf(x[4 * i + k], -e);
#pragma unroll
            for (int n = 0; n < 3; n++) {
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
                w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
                t[n][i] = w;
                y[0] -= __builtin_amdgcn_cvt_f32_fp8(w, 0);
                y[1] -= __builtin_amdgcn_cvt_f32_fp8(w, 1);
                y[2] -= __builtin_amdgcn_cvt_f32_fp8(w, 2);
                y[3] -= __builtin_amdgcn_cvt_f32_fp8(w, 3);
            }
        }
        return __builtin_amdgcn_ldexpf(1.f, e);
    }
    __device__ __forceinline__ float4_t times(const KPiece<uint8_t> (&k)[ND]) const
    {
        float4_t s = {0.f, 0.f, 0.f, 0.f};
        if constexpr (ND == 2) {
            i8_t a;
#pragma unroll
            for (int i = 0; i < 8; i++) a[i] = (int)k[i / 4].w[i & 3];
#pragma unroll
            for (int n = 2; n >= 0; n--) {
                i8_t b;
#pragma unroll
                for (int i = 0; i < 8; i++) b[i] = t[n][i];
                // (scales of 2^0: e8m0 127 in every byte)
                s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, s, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
            }
        } else {
#pragma unroll
            for (int n = 2; n >= 0; n--)
#pragma unroll
                for (int c = 0; c < 2; c++)
                    s = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8((long)((uint64_t)k[0].w[2 * c + 1] << 32 | k[0].w[2 * c]),
                                                                   (long)((uint64_t)(unsigned)t[n][2 * c + 1] << 32 | (unsigned)t[n][2 * c]), s, 0, 0, 0);
        }
        return s;
    }
};

// Eight keys by VD columns (8 or 4) of V, as loaded: a row of columns per key
template <class P, int VD>
struct VBlock;
template <int VD>
struct VBlock<uint8_t, VD> {
    unsigned w[8][VD / 4];
    __device__ __forceinline__ void load(int i, const uint8_t *p)
    {
        if constexpr (VD == 8) {
            const u2_t x = *reinterpret_cast<const u2_t *>(p);
            w[i][0] = x[0];
            w[i][1] = x[1];
        } else w[i][0] = *reinterpret_cast<const unsigned *>(p);
    }
    __device__ __forceinline__ void zero(int i)
    {
#pragma unroll
        for (int j = 0; j < VD / 4; j++) w[i][j] = 0;
    }
    __device__ __forceinline__ bool strip(int i)           // of its NaNs, whether there were any
    {
        bool any = false;
#pragma unroll
        for (int j = 0; j < VD / 4; j++) {
            const unsigned bad = ((w[i][j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            any = any || bad;
            w[i][j] &= ~((bad >> 7) * 0xffu);
        }
        return any;
    }
    __device__ __forceinline__ float value(int c) const    // of the first key
    {
        return (c & 3) == 0 ? __builtin_amdgcn_cvt_f32_fp8(w[0][c / 4], 0) : (c & 3) == 1 ? __builtin_amdgcn_cvt_f32_fp8(w[0][c / 4], 1)
             : (c & 3) == 2 ? __builtin_amdgcn_cvt_f32_fp8(w[0][c / 4], 2) : __builtin_amdgcn_cvt_f32_fp8(w[0][c / 4], 3);
    }
    // columns 2 c and 2 c + 1, each over the eight keys
    __device__ __forceinline__ void columns(int c, half8_t *a, half8_t *b) const
    {
        Frag x, y;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned k0 = cvt8(w[2 * i][c / 2], c & 1), k1 = cvt8(w[2 * i + 1][c / 2], c & 1);
            x.u[i] = __builtin_amdgcn_perm(k1, k0, 0x05040100u);
            y.u[i] = __builtin_amdgcn_perm(k1, k0, 0x07060302u);
        }
        *a = x.h;
        *b = y.h;
    }
};
template <int VD>
struct VBlock<half_t, VD> {
    unsigned w[8][VD / 2];
    __device__ __forceinline__ void load(int i, const half_t *p)
    {
        if constexpr (VD == 8) {
            const u4_t x = *reinterpret_cast<const u4_t *>(p);
#pragma unroll
            for (int j = 0; j < 4; j++) w[i][j] = x[j];
        } else {
            const u2_t x = *reinterpret_cast<const u2_t *>(p);
            w[i][0] = x[0];
            w[i][1] = x[1];
        }
    }
    __device__ __forceinline__ void zero(int i)
    {
#pragma unroll
        for (int j = 0; j < VD / 2; j++) w[i][j] = 0;
    }
    __device__ __forceinline__ bool strip(int i)           // of its NaNs and infinities, whether there were any
    {
        bool any = false;
#pragma unroll
        for (int j = 0; j < VD / 2; j++) {
            const unsigned low = (w[i][j] & 0x7c00u) == 0x7c00u ? 0xffffu : 0u, high = (w[i][j] & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u;
            any = any || (low | high);
            w[i][j] &= ~(low | high);
        }
        return any;
    }
    __device__ __forceinline__ float value(int c) const { return h2f(__builtin_bit_cast(half2_t, w[0][c / 2])[c & 1]); }
    __device__ __forceinline__ void columns(int c, half8_t *a, half8_t *b) const
    {
        Frag x, y;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x.u[i] = __builtin_amdgcn_perm(w[2 * i + 1][c], w[2 * i][c], 0x05040100u);
            y.u[i] = __builtin_amdgcn_perm(w[2 * i + 1][c], w[2 * i][c], 0x07060302u);
        }
        *a = x.h;
        *b = y.h;
    }
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// What the pages of a wave's positions are: where their rows of this head begin and what their scales make of a score
struct Entry {
    int64_t at[kEntries];
    float c[kEntries], lg[kEntries], iv[kEntries];         // alpha ks log2 e (more than 0), log2 vs, 1 / vs
};
struct Scales {
    float c, lg, iv;
};
// ... of page pg; pages of 16 bits have none
template <class P>
__device__ __forceinline__ Scales scales_of(const Entry &e, int pg, float alpha)
{
    if (sizeof(P) == 2) return {fmaxf(alpha * 1.44269504088896340736f, 1e-30f), 0.f, 1.f};
    return {e.c[pg], e.lg[pg], e.iv[pg]};
}

// The scores s of 32 positions of a lane's row (eight of them, in two registers of four) to weights: with c > 0 and lg of the
// lane's page, t = s c + lg.  Takes part in the running m and sum l (of weights by iv) and scales o where m grows; returns the
// weights in f16.  seen: how many of the lane's eight positions its row sees; edge (the same in all lanes): not all of all.
// SLACK: m grows only where a lane has more than kSlack above it, else the row's lanes need not hear of each other's scores; weights are
// 2^-kSlack of what they are otherwise, for they may be 2^kSlack too large (prompts in 16 bits of up to 900 rows and 4000 positions, 16
// heads of 128: 78.6 -> 74.1 us; single tokens, bound by memory, gain nothing).
constexpr float kTop = 15.f, kSlack = 8.f;
// x + a half of h, the conversion and the sum (in fp32) in one operation
__device__ __forceinline__ float plus_low(float x, unsigned h)
{
    asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "+v"(x) : "v"(h));
    return x;
}
__device__ __forceinline__ float plus_high(float x, unsigned h)
{
    asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(x) : "v"(h));
    return x;
}
template <bool SLACK, int N>
__device__ __forceinline__ half8_t weigh(float4_t (&s)[2], float c, float lg, float iv, float &m, float &l, float4_t (&o)[N], bool edge, int seen)
{
    if (edge) {
#pragma unroll
        for (int i = 0; i < 8; i++) s[i / 4][i & 3] = i < seen ? s[i / 4][i & 3] : -INFINITY;
    }
    float raw = s[0][0];                       // (c > 0: the largest of t is that of the largest of s)
#pragma unroll
    for (int i = 1; i < 8; i++) raw = fmaxf(raw, s[i / 4][i & 3]);
    const float mine = __builtin_fmaf(raw, c, lg);
    if (__ballot(mine > (SLACK ? m + kSlack : m))) {
        const float mn = fmaxf(m, with32(with16(mine, OpMax()), OpMax())), f = exp2_of(m - finite_max(mn));
        m = mn;
        l *= f;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] *= f;
    }
    const float off = lg + (SLACK ? kTop - kSlack : kTop) - finite_max(m);
    float even = 0.f, uneven = 0.f;
    Frag p;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float x = exp2_of(__builtin_fmaf(s[i / 2][2 * i & 3], c, off)), y = exp2_of(__builtin_fmaf(s[i / 2][(2 * i & 3) + 1], c, off));
        const half2_t pair = {f2h(x), f2h(y)};
        p.u[i] = __builtin_bit_cast(unsigned, pair);
        even = SLACK ? plus_low(even, p.u[i]) : even + x;
        uneven = SLACK ? plus_high(uneven, p.u[i]) : uneven + y;
    }
    l = __builtin_fmaf(even + uneven, iv, l);
    return p.h;
}

// One tile of rows and a part of its positions, by a wave.  ND: pieces of 64 columns of a head
template <int ND, int NR, class P>
struct Tile {
    static constexpr int VD = 4 * ND;          // columns of V of a lane
    const AttnArgs &a;
    Entry &entry;                              // the wave's, in LDS
    Query<ND, P> q[NR];                        // the lane's row of each 16: its query, a score's factor, its last position
    float factor[NR];
    int last[NR];
    float m[NR], l[NR];
    float4_t o[NR][VD];
    KPiece<P> kk[2][ND];
    VBlock<P, VD> vv;
    bool odd;                                  // there was a NaN or an infinity of V that some rows see

    __device__ __forceinline__ int page_of(int x) const { return shares::page_of(x, a.page_magic); }

    // keys and values of the 32 positions from x on, counted from the first entry's page; behind `end` the last one again
    __device__ __forceinline__ void load_k(int x, int end)
    {
        const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int j = min(x + 8 * (r16 >> 2) + 4 * t + (r16 & 3), end - 1), pg = page_of(j);
            const P *row = (const P *)a.k_pages + entry.at[pg] + __umul24(j - __umul24(pg, a.pb.page), a.Dp);
#pragma unroll
            for (int c = 0; c < ND; c++) {
                kk[t][c].load(row + min(64 * c + 16 * g, a.Dp - 16));
                // (there the query is zero, and an infinity of another column would make a NaN with it)
                if constexpr (sizeof(P) == 2)
                    if (64 * c + 16 * g >= a.Dp) kk[t][c].zero();
            }
        }
    }
    __device__ __forceinline__ void load_v(int x, int end)
    {
        const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
        const int j0 = x + 8 * g, pg = page_of(min(j0, end - 1));          // one page: of 16 positions or a multiple
        const P *row = (const P *)a.v_pages + entry.at[pg] + min(VD * r16, a.Dp - VD);
#pragma unroll
        for (int i = 0; i < 8; i++) vv.load(i, row + __umul24(min(j0 + i, end - 1) - __umul24(pg, a.pb.page), a.Dp));
    }

    // positions c0 .. c1 - 1 of rows row0 .. of sequence s
    __device__ __forceinline__ void run(int b, const Sequence &s, int h, int rows, int row0, int c0, int c1)
    {
        const int lane = lane_here(), r16 = lane & 15;
        odd = false;
        if (c0 >= c1) {                        // none of these positions is seen: nothing of them
#pragma unroll
            for (int n = 0; n < NR; n++) {
                m[n] = -INFINITY;
                l[n] = 0.f;
#pragma unroll
                for (int i = 0; i < VD; i++) o[n][i] = float4_t{0.f, 0.f, 0.f, 0.f};
            }
            return;
        }
        const int least = uniform(s.first + row0 / a.G);       // positions up to there are seen by every row
        int base, end;
        float ks = 1.f, vs = 1.f;
        // the pages from position `seg` on: their numbers, their addresses and the first keys and values, what their scales make
        auto look_up = [&](int seg) __attribute__((always_inline)) {
            const Pages p(uniform(seg), c1, a.pb.page);
            base = p.base;
            end = p.end;
            return a.pb.table[(int64_t)b * a.pb.ldt + p.p0 + min(lane, p.last(a.page_magic))];
        };
        auto request = [&](int id, int x) __attribute__((always_inline)) {
            if (id < 0 || id >= a.pb.P) {
                report(a.pb, b);
                id = 0;                        // its rows are unspecified, not its reads
            }
            const int64_t ph = (int64_t)id * a.Hkv + h;
            if (sizeof(P) == 1) ks = a.k_scale[ph], vs = a.v_scale[ph];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");         // (the entries of before are done with)
            __builtin_amdgcn_wave_barrier();
            entry.at[lane] = ph * a.pb.page * a.Dp;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            load_k(x, end);
            load_v(x, end);
        };
        auto scales = [&]() __attribute__((always_inline)) {
            entry.c[lane] = fmaxf(ks * (a.alpha * 1.44269504088896340736f), 1e-30f);
            entry.lg[lane] = __builtin_amdgcn_logf(vs);
            entry.iv[lane] = __builtin_amdgcn_rcpf(vs);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };
        {
            const int id = look_up(c0);
            QueryWords<ND> words[NR];          // requested with the pages' numbers
#pragma unroll
            for (int n = 0; n < NR; n++) {
                const int r = min(row0 + 16 * n + r16, rows - 1), t = r / a.G;
                last[n] = s.first + t;
                words[n].load(a.q + (int64_t)(s.s0 + t) * a.ldq + (h * a.G + r - t * a.G) * a.Dh, a.Dh, lane >> 4);
            }
            request(id, c0 - base);
#pragma unroll
            for (int n = 0; n < NR; n++) factor[n] = q[n].set(words[n], a.Dh, a.sign);
            scales();
        }
#pragma unroll
        for (int n = 0; n < NR; n++) {
            m[n] = -INFINITY;
            l[n] = 0.f;
#pragma unroll
            for (int i = 0; i < VD; i++) o[n][i] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        for (int x = c0 - base;;) {
            for (; x < end; x += kStep) step(x, end, least - base, base, min(x + kStep, end - 1));
            const int seg = base + end;
            if (seg >= c1) break;
            const int id = look_up(seg);
            x = seg - base;
            request(id, x);
            scales();
        }
    }

    __device__ __forceinline__ void step(int x, int end, int least, int base, int next)
    {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const bool edge = x + kStep - 1 > min(least, end - 1);             // some of these 32 positions are hidden from some row
        float4_t sc[NR][2];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int n = 0; n < NR; n++) sc[n][t] = q[n].times(kk[t]);
        load_k(next, end);
        const int pg = page_of(min(x + 8 * g, end - 1));       // of the lane's eight keys
        const Scales sc8 = scales_of<P>(entry, pg, a.alpha);
        half8_t w[NR];
#pragma unroll
        for (int n = 0; n < NR; n++)
            w[n] = weigh<false>(sc[n], sc8.c * factor[n], sc8.lg, sc8.iv, m[n], l[n], o[n], edge, min(last[n] - base, end - 1) - (x + 8 * g) + 1);
        if (edge) {
            // what no row of the tile sees is nothing; a NaN or an infinity that some rows see must not meet the zero weights of
            // the others: it is added at the end
            bool any = false;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int j = x + 8 * g + i;
                if (j >= end) vv.zero(i);
                else if (j > least) any = vv.strip(i) || any;
            }
            if (__ballot(any)) odd = true;
        }
#pragma unroll
        for (int c = 0; c < VD / 2; c++) {
            half8_t v0, v1;
            vv.columns(c, &v0, &v1);
#pragma unroll
            for (int n = 0; n < NR; n++) {
                o[n][2 * c] = mfma(v0, w[n], o[n][2 * c]);
                o[n][2 * c + 1] = mfma(v1, w[n], o[n][2 * c + 1]);
            }
            __builtin_amdgcn_sched_barrier(0);             // (all of V turned at once is 64 registers)
        }
        load_v(next, end);
    }

    // NaNs and infinities of V at positions j0 .. j1 - 1, each to the rows that see it
    __device__ __forceinline__ void add_odd(int b, int h, int j0, int j1)
    {
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll 1
        for (int j = j0; j < j1; j++) {
            const int id = a.pb.table[(int64_t)b * a.pb.ldt + j / a.pb.page];
            const P *v = (const P *)a.v_pages + (((int64_t)(id < 0 || id >= a.pb.P ? 0 : id) * a.Hkv + h) * a.pb.page + j % a.pb.page) * a.Dp;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                VBlock<P, VD> x;
                x.load(0, v + min(VD * (4 * g + i), a.Dp - VD));
#pragma unroll
                for (int c = 0; c < VD; c++)
#pragma unroll
                    for (int n = 0; n < NR; n++)
                        if (!(fabsf(x.value(c)) < INFINITY) && j <= last[n]) o[n][c][i] += x.value(c);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // What other waves of the workgroup have of the tile, through LDS
    struct Deposit {
        float4_t o[NR][VD][64];
        float m[NR][64], l[NR][64];
    };
    __device__ __forceinline__ void put(Deposit &to) const
    {
        const int lane = lane_here();
#pragma unroll
        for (int n = 0; n < NR; n++) {
            to.m[n][lane] = m[n];
            to.l[n][lane] = l[n];
#pragma unroll
            for (int c = 0; c < VD; c++) to.o[n][c][lane] = o[n][c];
        }
    }
    __device__ __forceinline__ void add(const Deposit &x)
    {
        const int lane = lane_here();
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const float mx = x.m[n][lane], mn = fmaxf(m[n], mx), origin = finite_max(mn), f = exp2_of(m[n] - origin), fx = exp2_of(mx - origin);
            m[n] = mn;
            l[n] = l[n] * f + x.l[n][lane] * fx;
#pragma unroll
            for (int c = 0; c < VD; c++) o[n][c] = o[n][c] * f + x.o[n][c][lane] * fx;
        }
    }

    // A lane has columns VD (4 g + i) + c of its row in o[.][c][i].  slot < 0: to the output
    __device__ __forceinline__ void write(const Sequence &s, int h, int rows, int row0, int slot)
    {
        const int lane = lane_here(), r16 = lane & 15, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const float sum = with32(with16(l[n], OpSum()), OpSum());
            const int r = row0 + 16 * n + r16, t = r / a.G;
            if (r >= rows) continue;
            const float y = slot >= 0 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
            const int64_t at = (int64_t)slot * (16 * NR) + 16 * n + r16;
            half_t *out = a.out + (int64_t)(s.s0 + t) * a.ldo + (h * a.G + r - t * a.G) * a.Dh;
            float *part = a.part + at * a.Dh;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int c = 0; c < VD; c += 4) {
                    const int d = VD * (4 * g + i) + c;
                    if (d >= a.Dh) continue;
                    const float4_t v = {o[n][c][i] * y, o[n][c + 1][i] * y, o[n][c + 2][i] * y, o[n][c + 3][i] * y};
                    if (slot >= 0) *reinterpret_cast<float4_t *>(part + d) = v;
                    else *reinterpret_cast<half4_t *>(out + d) = half4_t{f2h(v[0]), f2h(v[1]), f2h(v[2]), f2h(v[3])};
                }
            if (slot >= 0 && g == 0) {
                a.stats[2 * at] = m[n];
                a.stats[2 * at + 1] = sum;
            }
        }
    }
};

// Waves of a SIMD: as many as the registers are for
constexpr int resident(int ND, int NR, int bytes) { return NR == 1 && ND * bytes < 4 ? 3 : 2; }

template <int ND, int NR, class P>
__global__ void __launch_bounds__(kThreads, resident(ND, NR, sizeof(P))) paged_attention_kernel(AttnArgs a)
{
    constexpr int kRows = 16 * NR;
    __shared__ Entry entries[kWaves];
    __shared__ typename Tile<ND, NR, P>::Deposit deposits[kWaves - 1];     // of waves 1, 2, 3
    const unsigned wid = uniform((int)threadIdx.x >> 6), group = blockIdx.x;
    const Sequence s64 = lane_sequence(a, 0);              // of the first 64 sequences, which mostly are all
    const double u64 = share_of(a, kRows, s64).units;      // (whole numbers)
    double all = u64;
    for (int b0 = 64; b0 < a.pb.B; b0 += 64) all += share_of(a, kRows, lane_sequence(a, b0)).units;
    all = wave_sum_f64(all);
    if (too_much(all)) return;
    const unsigned units = uniform((int)(unsigned)all), groups = groups_of(a.groups, units);
    if (group >= groups) return;
    const Shares shares(units, groups);
    const unsigned x0 = uniform((int)shares.begin(group)), x1 = uniform((int)shares.begin(group + 1));     // the workgroup's
    auto begin = [&](unsigned w) { return x0 + (x1 - x0) * w / kWaves; };  // and a wave's
    unsigned x = begin(wid);
    const unsigned until = begin(wid + 1);
    // the sequence in whose work x lies, and what there is before it
    int b = 0;
    unsigned before = 0;
    for (int b0 = 0; b0 < a.pb.B; b0 += 64) {
        const double u = b0 == 0 ? u64 : share_of(a, kRows, lane_sequence(a, b0)).units, upto = scan_f64(u) + (double)before;
        const uint64_t hit = __ballot(upto > (double)x);
        const int at = hit ? __ffsll((unsigned long long)hit) - 1 : 63;
        before = (unsigned)uniform((int)(unsigned)lane_f64(hit ? upto - u : upto, at));
        if (hit) {
            b = b0 + at;
            break;
        }
    }
    // Of a tile the workgroup has units g0 .. g1 - 1, this wave u0 .. u1 - 1.  The wave that has the first of them puts them together.
    Tile<ND, NR, P> t{a, entries[wid]};
    Sequence s;
    int h, row0, slot;
    unsigned g1 = 0;
    bool others = false;                       // there are other waves' to put together with what t has
    for (; x < until; b++) {
        s = b < 64 ? of_lane(s64, b) : sequence(a.pb, b, (int64_t)a.pb.W * a.pb.page, a.max_new);
        const Share w = share_of(a, kRows, s);
        const unsigned behind = before + w.units;
        while (x < until && x < behind) {
            const Part p(w, kRows, before, x, until, x0, x1);
            const int rows = s.n * a.G;
            h = p.h;
            row0 = p.row0;
            g1 = p.g1;
            x = p.u1;
            if (p.u1 <= p.u0) continue;        // (a share may end before the tile's first step)
            const int seen = uniform(s.first + min(rows - 1, row0 + kRows - 1) / a.G + 1);     // positions that some row sees
            const int c0 = p.c0(), c1 = p.c1(seen);
            const bool mine = p.u0 == p.g0;    // else it goes to the wave that has the tile's first
            slot = p.slot(group);
            others = mine && p.u1 < g1;
            t.run(b, s, h, rows, row0, c0, c1);
            if (t.odd) t.add_odd(b, h, max(c0, s.first + row0 / a.G + 1), c1);
            if (!mine) t.put(deposits[wid - 1]);
            else if (!others) t.write(s, h, rows, row0, slot);
        }
        before = behind;
    }
    __syncthreads();
    if (!others) return;
    for (unsigned w = wid + 1; w < kWaves && begin(w) < g1; w++)
        if (begin(w) < begin(w + 1)) t.add(deposits[w - 1]);
    t.write(s, h, s.n * a.G, row0, slot);
}

// ---------------------------------------------------------------- prompts
// Sequences with many new rows: 128 of them (tokens by the query heads of a key head) to a workgroup, 32 to each of its four waves,
// 64 positions at a time, whose keys and values go through LDS as f16: converted and V turned once for all waves (two of them
// see to the keys, two to the values), while the products of the 64 before them run, in two buffers with one barrier a step.
// 16-byte pieces of LDS rows are swapped by f(row), which spreads the sixteen rows of an operand, and the rows that a wave writes,
// evenly over the banks.  (16 rows to each of eight waves read the operands twice as often and have half the registers: 88.6
// against 83 us for three sequences of up to 900 rows and 4000 positions, 16 heads of 128, which are 71.5 us now, in 8 bits 73; one of 900
// and 24 single tokens of 1000 to 4000 in 8 bits 99, 39 of them the prompt's launch and 46 the tokens' behind it.)
//
// Shares are cut as above, a workgroup to a share and by steps of 64.  Workgroups of an XCD have neighbouring shares: the tiles of a
// head read its keys and values from one L2.
__device__ __forceinline__ int swap_of(int row) { return ((row >> 2) ^ row) & 7; }

constexpr int kBigThreads = 256, kBigWaves = kBigThreads / 64;

template <int ND, class P>
struct Prompt {
    static constexpr int NS = 2 * ND;          // matrix instructions along the columns of a key
    static constexpr int kHalf = kBigThreads / 2;                          // lanes that load keys, and that load values
    static constexpr int kPer = 64 * ND * (int)sizeof(P) / 16;             // 16-byte pieces of a key
    static constexpr int kPieces = kBig * kPer / kHalf;                    // of a lane
    static constexpr int kApart = kHalf / kPer;                            // keys from one to the next
    static constexpr int kCols = 16 * ND;                                  // lanes that have a key's columns, four each, of V
    static constexpr int kBlocks = ND, kKeys = kBig / kBlocks;             // blocks of V of a lane, kKeys positions apart
    struct Shared {
        half_t k[2][kBig][64 * ND], v[2][64 * ND][kBig];
        Entry entry;
        int odd;
    };
    const AttnArgs &a;
    Shared &sh;
    half8_t q[2][NS];
    int last[2];
    float m[2], l[2];
    float4_t o[2][4 * ND];
    // the next 64 positions, as they come: keys (waves 2 and 3) or values
    union {
        u4_t k[kPieces];
        VBlock<P, 4> v[kBlocks];
    } next;

    __device__ __forceinline__ int page_of(int x) const { return shares::page_of(x, a.page_magic); }

    // 16 positions in a row are of one page (x: the first of them, of full ones), and so is all that a wave loads at once: the address
    // of its first row is a scalar, a lane's part of it the same every time (but for the positions behind `end`).
    __device__ __forceinline__ const char *page_at(const void *pages, int x) const
    {
        const int pg = uniform((int)((unsigned)x * a.page_magic >> 22));
        const int64_t at = sh.entry.at[pg];
        const uint64_t first = (uint64_t)(unsigned)uniform((int)(at >> 32)) << 32 | (unsigned)uniform((int)at);
        return (const char *)pages + (first + (unsigned)((x - pg * a.pb.page) * a.Dp)) * sizeof(P);
    }
    // What of the addresses is a lane's own: its row and columns in memory, bytes from the wave's first row, and its place in
    // LDS, halves from a buffer's start (keys: of the first piece; values: of column 0 of 4)
    struct Own {
        unsigned from;
        int to;
    };
    __device__ __forceinline__ Own own() const
    {
        const int tid = threadIdx.x & (kHalf - 1), lane = tid & 63;
        Own w;
        if (threadIdx.x >= kHalf) {
            w.from = (__umul24(lane / kPer, a.Dp) + min(lane % kPer * (16 / (int)sizeof(P)), a.Dp - 16 / (int)sizeof(P))) * (unsigned)sizeof(P);
            const int j = tid / kPer, c = tid % kPer * (16 / (int)sizeof(P)) / 8;
            w.to = j * 64 * ND + (c ^ swap_of(j)) * 8;
        } else {
            w.from = (__umul24((8 * (lane / kCols)) & 15, a.Dp) + min(4 * (lane % kCols), a.Dp - 4)) * (unsigned)sizeof(P);
            const int kg = tid / kCols, d = 4 * (tid % kCols);
            w.to = d * kBig + (kg ^ swap_of(d)) * 8;
        }
        return w;
    }
    __device__ __forceinline__ void load(const Own &w, int x, int end)
    {
        const int wid = uniform((int)threadIdx.x >> 6);
        if (wid >= kBigWaves / 2) {
            const int first = 64 * (wid - kBigWaves / 2) / kPer;
            if (x + kBig <= end) {
                const char *before = nullptr;
#pragma unroll
                for (int i = 0; i < kPieces; i++) {    // (kApart: 8, two pieces to 16 positions, or a multiple of 16)
                    const char *k = kApart < 16 && (i & 1) ? nullptr
                                                           : page_at(a.k_pages, x + (first & ~15) + i * kApart) + (first & 15) * a.Dp * (int)sizeof(P);
                    if (kApart < 16 && (i & 1)) k = before + kApart * a.Dp * (int)sizeof(P);
                    next.k[i] = *reinterpret_cast<const u4_t *>(k + w.from);
                    before = k;
                }
                return;
            }
            const int lane = lane_here();
#pragma unroll
            for (int i = 0; i < kPieces; i++) {
                const int j = min(x + first + i * kApart + lane / kPer, end - 1), pg = page_of(j);
                const P *row = (const P *)a.k_pages + sh.entry.at[pg] + __umul24(j - __umul24(pg, a.pb.page), a.Dp);
                next.k[i] = *reinterpret_cast<const u4_t *>(row + min(lane % kPer * (16 / (int)sizeof(P)), a.Dp - 16 / (int)sizeof(P)));
            }
        } else {
            const int first = 8 * (64 / kCols) * wid;          // 16 positions to a wave or, ND 1, 32
            if (x + kBig <= end) {
#pragma unroll
                for (int k = 0; k < kBlocks; k++) {
                    const char *v = page_at(a.v_pages, x + first + k * kKeys);
                    if (ND == 1) {
                        const char *v1 = page_at(a.v_pages, x + first + 16);
                        v = (threadIdx.x & 32) ? v1 : v;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) next.v[k].load(i, (const P *)(v + i * a.Dp * (int)sizeof(P) + w.from));
                }
                return;
            }
            const int lane = lane_here();
#pragma unroll
            for (int k = 0; k < kBlocks; k++) {
                const int j0 = x + first + k * kKeys + 8 * (lane / kCols), pg = page_of(min(j0, end - 1));
                const P *row = (const P *)a.v_pages + sh.entry.at[pg] + min(4 * (lane % kCols), a.Dp - 4);
#pragma unroll
                for (int i = 0; i < 8; i++) next.v[k].load(i, row + __umul24(min(j0 + i, end - 1) - __umul24(pg, a.pb.page), a.Dp));
            }
        }
    }
    // ... into buffer `to`; least: positions up to there are seen by every row of the tile
    __device__ __forceinline__ void store(const Own &own, int to, int x, int end, int least)
    {
        const int wid = uniform((int)threadIdx.x >> 6);
        half_t *kb = &sh.k[to][0][0], *vb = &sh.v[to][0][0];
        if (wid >= kBigWaves / 2) {
            if ((threadIdx.x & 63) % kPer * (16 / (int)sizeof(P)) >= a.Dp) // (beside the columns the queries are zeros, and so must the keys be)
#pragma unroll
                for (int i = 0; i < kPieces; i++) next.k[i] = u4_t{0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < kPieces; i++)
#pragma unroll
                for (int k = 0; k < 16 / (int)sizeof(P) / 8; k++) {
                    Frag f;
#pragma unroll
                    for (int w = 0; w < 4; w++) f.u[w] = sizeof(P) == 2 ? next.k[i][w] : cvt8(next.k[i][2 * k + w / 2], w & 1);
                    *reinterpret_cast<half8_t *>(kb + (own.to ^ (8 * k) ^ 8 * (i * kApart / 4 & 7)) + i * kApart * 64 * ND) = f.h;
                }
        } else {
#pragma unroll
            for (int b = 0; b < kBlocks; b++) {
                VBlock<P, 4> &v = next.v[b];
                if (x + kBig - 1 > min(least, end - 1)) {
                    const int j0 = x + b * kKeys + 8 * ((64 * wid + lane_here()) / kCols);
                    bool any = false;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if (j0 + i >= end) v.zero(i);
                        else if (j0 + i > least) any = v.strip(i) || any;
                    }
                    if (any) sh.odd = 1;
                }
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    half8_t v0, v1;
                    v.columns(c, &v0, &v1);
                    *reinterpret_cast<half8_t *>(vb + (own.to ^ b * kKeys ^ (16 * c)) + 2 * c * kBig) = v0;            // swap_of(d + e) = swap_of(d) ^ e
                    *reinterpret_cast<half8_t *>(vb + (own.to ^ b * kKeys ^ (16 * c + 8)) + (2 * c + 1) * kBig) = v1;
                }
            }
        }
    }

    // Where a lane reads its operands, in halves from the start of a buffer.  A key's row is j = 32 b + 8 (r16 / 4) + 4 t + r16 % 4,
    // so swap_of(j) = 2 (r16 / 4) ^ r16 % 4 ^ 5 t; a row of V is d = 16 c + r16, swap_of(d) = r16 / 4 ^ r16 & 7 ^ 4 (c & 1).  The
    // lane's place with b, c and t all 0; these swaps turn bits of it, the rest is a constant of the instruction.
    struct Places {
        int k, v;
    };
    __device__ __forceinline__ Places places() const
    {
        const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4, a4 = r16 >> 2, b4 = r16 & 3;
        return {(8 * a4 + b4) * 64 * ND + (g ^ (2 * a4) ^ b4) * 8, r16 * kBig + (g ^ ((a4 ^ r16) & 7)) * 8};
    }

    // 32 positions, those from x on, block b of the buffer; least: positions up to there are seen by every row of the wave
    __device__ __forceinline__ void step(const Places &at, int from, int b, int x, int end, int base, int least)
    {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const half_t *kb = &sh.k[from][0][0] + 32 * b * 64 * ND, *vb = &sh.v[from][0][0];
        float4_t sc[2][2] = {};
#pragma unroll
        for (int c = 0; c < NS; c++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const half8_t k = *reinterpret_cast<const half8_t *>(kb + (at.k ^ (40 * t) ^ (32 * (c & 1))) + 4 * t * 64 * ND + (c >> 1) * 64);
#pragma unroll
                for (int n = 0; n < 2; n++) sc[n][t] = mfma(k, q[n][c], sc[n][t]);
            }
        const int v0 = at.v ^ (32 * b);
        half8_t vf[4];                         // four operands ahead (one by one, waited for: 87 against 83 us)
#pragma unroll
        for (int c = 0; c < 4; c++) vf[c] = *reinterpret_cast<const half8_t *>(vb + (v0 ^ (32 * (c & 1))) + 16 * c * kBig);
        const int pg = page_of(min(x + 8 * g, end - 1));
        const Scales sc8 = scales_of<P>(sh.entry, pg, a.alpha);
        const bool edge = x + 31 > min(least, end - 1);
        half8_t p[2];
#pragma unroll
        for (int n = 0; n < 2; n++)
            p[n] = weigh<sizeof(P) == 2>(sc[n], sc8.c, sc8.lg, sc8.iv, m[n], l[n], o[n], edge, min(last[n] - base, end - 1) - (x + 8 * g) + 1);
#pragma unroll
        for (int c = 0; c < 4 * ND; c++) {
#pragma unroll
            for (int n = 0; n < 2; n++) o[n][c] = mfma(vf[c & 3], p[n], o[n][c]);
            if (c + 4 < 4 * ND) vf[c & 3] = *reinterpret_cast<const half8_t *>(vb + (v0 ^ (32 * (c & 1))) + 16 * (c + 4) * kBig);
        }
#pragma unroll
        for (int c = 0; c < 4 * ND - 4; c++) {             // (two matrix instructions, one read)
            __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 8, 0);
    }

    // positions c0 .. c1 - 1 of rows row0 .. of sequence s; none where a share is behind the last that is seen (c1 > 0)
    __device__ __forceinline__ void run(int b, const Sequence &s, int h, int rows, int row0, int c0, int c1)
    {
        const int wid = uniform((int)threadIdx.x >> 6), lane = lane_here(), tid = 64 * wid + lane, r16 = lane & 15, g = lane >> 4;
        const int mine = row0 + 32 * wid;      // the wave's first row
        // the pages from position `seg` on: the lane's number of them
        auto look_up = [&](int seg) __attribute__((always_inline)) {
            const Pages p(uniform(seg), c1, a.pb.page);
            return a.pb.table[(int64_t)b * a.pb.ldt + p.p0 + min(lane, p.last(a.page_magic))];
        };
        int id = look_up(BigPart::look(c0, c1));           // requested with the queries
        u2_t words[2][2 * NS];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int r = min(mine + 16 * n + r16, rows - 1), t = r / a.G;
            last[n] = s.first + t;
            const half_t *qr = a.q + (int64_t)(s.s0 + t) * a.ldq + (h * a.G + r - t * a.G) * a.Dh;
#pragma unroll
            for (int c = 0; c < 2 * NS; c++) words[n][c] = *reinterpret_cast<const u2_t *>(qr + min(32 * (c / 2) + 8 * g + 4 * (c & 1), a.Dh - 4));
        }
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int c = 0; c < NS; c++) {
                Frag f;
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const bool there = 32 * c + 8 * g + 4 * j < a.Dh;
                    f.u[2 * j] = there ? words[n][2 * c + j][0] ^ a.sign : 0u;
                    f.u[2 * j + 1] = there ? words[n][2 * c + j][1] ^ a.sign : 0u;
                }
                q[n][c] = f.h;
            }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            m[n] = -INFINITY;
            l[n] = 0.f;
#pragma unroll
            for (int i = 0; i < 4 * ND; i++) o[n][i] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
        const int least = uniform(s.first + row0 / a.G);                               // seen by every row of the tile
        const int wave_least = uniform(s.first + min(mine, rows - 1) / a.G), wave_last = uniform(mine < rows ? s.first + (min(mine + 32, rows) - 1) / a.G : -1);
        const Places at = places();
        const Own w = own();
        for (int seg = c0; seg < c1;) {
            const Pages pages(uniform(seg), c1, a.pb.page);
            const int base = pages.base, end = pages.end;
            __syncthreads();                   // (entries and buffers of before are done with)
            if (seg != c0) id = look_up(seg);
            if (tid < 64) {
                if (id < 0 || id >= a.pb.P) {
                    report(a.pb, b);
                    id = 0;                    // its rows are unspecified, not its reads
                }
                const int64_t ph = (int64_t)id * a.Hkv + h;
                float ks = 1.f, vs = 1.f;
                if (sizeof(P) == 1) ks = a.k_scale[ph], vs = a.v_scale[ph];
                sh.entry.at[lane] = ph * a.pb.page * a.Dp;
                sh.entry.c[lane] = fmaxf(ks * (a.alpha * 1.44269504088896340736f), 1e-30f);
                sh.entry.lg[lane] = __builtin_amdgcn_logf(vs);
                sh.entry.iv[lane] = __builtin_amdgcn_rcpf(vs);
                if (seg == c0 && lane == 0) sh.odd = 0;
            }
            __syncthreads();
            int x = seg - base, buffer = 0;
            load(w, x, end);
            store(w, 0, x, end, least - base);
            __syncthreads();
            for (; x < end; x += kBig) {
                const bool more = x + kBig < end;
                load(w, more ? x + kBig : x, end);
#pragma unroll
                for (int half = 0; half < 2; half++)
                    if (x + 32 * half <= min(wave_last - base, end - 1)) step(at, buffer, half, x + 32 * half, end, base, wave_least - base);
                buffer ^= 1;
                if (more) store(w, buffer, x + kBig, end, least - base);
                __syncthreads();
            }
            seg = base + end;
        }
    }

    __device__ __forceinline__ void write(int b, const Sequence &s, int h, int rows, int row0, int c0, int c1, int slot)
    {
        const int lane = lane_here(), wid = uniform((int)threadIdx.x >> 6), r16 = lane & 15, g = lane >> 4;
        if (c0 < c1 && sh.odd) {               // NaNs and infinities of V, each to the rows that see it
#pragma unroll 1
            for (int j = max(c0, s.first + row0 / a.G + 1); j < c1; j++) {
                const int id = a.pb.table[(int64_t)b * a.pb.ldt + j / a.pb.page];
                const P *v = (const P *)a.v_pages + (((int64_t)(id < 0 || id >= a.pb.P ? 0 : id) * a.Hkv + h) * a.pb.page + j % a.pb.page) * a.Dp;
#pragma unroll
                for (int c = 0; c < 4 * ND; c++) {
                    VBlock<P, 4> x;
                    x.load(0, v + min(16 * c + 4 * g, a.Dp - 4));
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int n = 0; n < 2; n++)
                            if (!(fabsf(x.value(i)) < INFINITY) && j <= last[n]) o[n][c][i] += x.value(i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const float sum = with32(with16(l[n], OpSum()), OpSum());
            const int r = row0 + 32 * wid + 16 * n + r16, t = r / a.G;
            if (r >= rows) continue;
            const float y = slot >= 0 ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
            const int64_t at = (int64_t)slot * kPrompt + r - row0;
            half_t *out = a.out + (int64_t)(s.s0 + t) * a.ldo + (h * a.G + r - t * a.G) * a.Dh;
            float *part = a.big_part + at * a.Dh;
#pragma unroll
            for (int c = 0; c < 4 * ND; c++) {
                const int d = 16 * c + 4 * g;
                if (d >= a.Dh) continue;
                const float4_t v = o[n][c] * y;
                if (slot >= 0) *reinterpret_cast<float4_t *>(part + d) = v;
                else *reinterpret_cast<half4_t *>(out + d) = half4_t{f2h(v[0]), f2h(v[1]), f2h(v[2]), f2h(v[3])};
            }
            if (slot >= 0 && g == 0) {
                a.big_stats[2 * at] = m[n];
                a.big_stats[2 * at + 1] = sum;
            }
        }
    }
};

template <int ND, class P>
__global__ void __launch_bounds__(kBigThreads, 2) paged_prompt_kernel(AttnArgs a)
{
    __shared__ typename Prompt<ND, P>::Shared sh;
    const int lane = threadIdx.x & 63;
    const Sequence s64 = lane_sequence(a, 0);
    const double u64 = big_share_of(a, s64).units(a.Hkv);
    double all = u64;
    for (int b0 = 64; b0 < a.pb.B; b0 += 64) all += big_share_of(a, lane_sequence(a, b0)).units(a.Hkv);
    all = wave_sum_f64(all);
    if (too_much(all)) return;
    const unsigned units = uniform((int)(unsigned)all), groups = big_groups_of(a.big_groups, units);
    const unsigned group = xcd_order(blockIdx.x, a.big_groups);
    if (units == 0 || group >= groups) return;
    const Shares shares(units, groups);
    unsigned x = uniform((int)shares.begin(group));
    const unsigned until = uniform((int)shares.begin(group + 1));
    int b = 0;
    unsigned before = 0;
    for (int b0 = 0; b0 < a.pb.B; b0 += 64) {
        const double u = b0 == 0 ? u64 : big_share_of(a, lane_sequence(a, b0)).units(a.Hkv), upto = scan_f64(u) + (double)before;
        const uint64_t hit = __ballot(upto > (double)x);
        const int at = hit ? __ffsll((unsigned long long)hit) - 1 : 63;
        before = (unsigned)uniform((int)(unsigned)lane_f64(hit ? upto - u : upto, at));
        if (hit) {
            b = b0 + at;
            break;
        }
    }
    for (; x < until; b++) {
        const Sequence s = b < 64 ? of_lane(s64, b) : sequence(a.pb, b, (int64_t)a.pb.W * a.pb.page, a.max_new);
        const BigShare w = big_share_of(a, s);
        const unsigned head = w.before(w.tiles), behind = before + w.units(a.Hkv);
        while (x < until && x < behind) {
            const int h = uniform((int)((x - before) / head)), rows = s.n * a.G;
            const unsigned in = x - before - h * head;
            int tile = 0;                  // that unit `in` of the head lies in
            for (int t0 = 0; t0 < w.tiles; t0 += 64) {
                const int n = __popcll(__ballot(t0 + lane < w.tiles && w.before(t0 + lane + 1) <= in));
                tile += n;
                if (n < 64) break;
            }
            tile = uniform(tile);
            const unsigned start = uniform((int)w.before(tile)), whole = uniform((int)w.before(tile + 1)) - start;
            const int from = (int)(in - start), to = (int)min(whole, from + (until - x)), row0 = tile * kPrompt;
            const int end = uniform(s.first + min(rows - 1, row0 + kPrompt - 1) / a.G + 1);
            const BigPart p(from, to, (int)whole);
            if (p.behind > p.first) {
                const int c0 = uniform(p.c0()), c1 = uniform(p.c1(end));
                Prompt<ND, P> t{a, sh};
                t.run(b, s, h, rows, row0, c0, c1);
                t.write(b, s, h, rows, row0, c0, c1, p.slot(group));
            }
            x += to - from;
        }
        before = behind;
    }
}

// Where the parts of a tile of rows are
__device__ __forceinline__ Parts parts_of(const AttnArgs &a, const Sequence &s, int rows, int h, int tile, unsigned units, unsigned before)
{
    unsigned first, steps, groups;
    if (s.n * a.G > a.few) {
        const BigShare w = big_share_of(a, s);
        first = before + h * w.before(w.tiles) + w.before(tile) + kBigBegin;
        steps = w.before(tile + 1) - w.before(tile) - kBigBegin;
        groups = big_groups_of(a.big_groups, units);
    } else {
        const Share w = share_of(a, rows, s);
        first = before + (unsigned)(h * w.tiles + tile) * (w.steps + begin_of(rows)) + begin_of(rows);
        steps = w.steps;
        groups = groups_of(a.groups, units);
    }
    Parts p(units, groups, first, steps);
    p.i0 = uniform(p.i0);
    p.count = uniform(p.count);
    return p;
}

// Parts put together as they come: maximum and sum of weights, and the weighted sums of N columns
template <int N>
struct Joined {
    float m = -INFINITY, l = 0.f, o[N] = {};
    // `AT` parts (m, l, o) at once; `there`: how many of them there are
    template <int AT>
    __device__ __forceinline__ void add(const float2 (&st)[AT], const float (&v)[AT][N], int there)
    {
        float mn = m;
#pragma unroll
        for (int k = 0; k < AT; k++) mn = k < there ? fmaxf(mn, st[k].x) : mn;
        const float origin = finite_max(mn), f = exp2_of(m - origin);
        m = mn;
        l *= f;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] *= f;
#pragma unroll
        for (int k = 0; k < AT; k++) {
            if (k >= there) continue;
            const float fk = exp2_of(st[k].x - origin);
            l = __builtin_fmaf(st[k].y, fk, l);
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = __builtin_fmaf(v[k][i], fk, o[i]);
        }
    }
};

// The parts of a row put together, two columns per lane, by a wave or, for few rows, a workgroup of four waves; zeros for rows whose
// sequence's numbers do not fit together, which the last workgroup names.  Bound by latency: eight parts are requested at once, their
// sums with their values.
template <int NR, int WAVES>
__global__ void __launch_bounds__(kThreads) paged_attention_join_kernel(AttnArgs a)
{
    constexpr int kRows = 16 * NR, kAtOnce = 8;
    const PagedBatch &pb = a.pb;
    const int lane = threadIdx.x & 63, wid = uniform((int)threadIdx.x >> 6), at_row = (int)blockIdx.x * (kWaves / WAVES) + (WAVES == 1 ? wid : 0);
    const int row = at_row / a.H, head = at_row - row * a.H, first = WAVES == 1 ? 0 : wid, d = min(2 * lane, a.Dh - 2);
    if (blockIdx.x == gridDim.x - 1) {         // names what does not fit, whether it has rows or not
        for (int b = threadIdx.x; b < pb.B; b += kThreads)
            if (!sequence(pb, b, (int64_t)pb.W * pb.page, a.max_new).ok) report(pb, b);
        return;
    }
    // all work, that of the sequences before the row's, and the row's sequence
    double all = 0., some = 0.;
    Sequence s = {0, 0, 0, false};
    int b = -1;
    for (int b0 = 0; b0 < pb.B; b0 += 64) {
        const Sequence q = lane_sequence(a, b0);
        const double u = share_of(a, kRows, q).units;
        const uint64_t hit = __ballot(b0 + lane < pb.B && row >= q.s0 && row < (int)((unsigned)q.s0 + (unsigned)q.n));
        all += u;
        some += b < 0 && (!hit || lane < __ffsll((unsigned long long)hit) - 1) ? u : 0.;
        if (hit && b < 0) {
            const int at = __ffsll((unsigned long long)hit) - 1;
            b = b0 + at;
            s = of_lane(q, at);
        }
    }
    if (b < 0 || row >= pb.T) return;
    half_t *out = a.out + row * a.ldo + head * a.Dh + d;
    if (!s.ok) {
        if (first == 0 && 2 * lane < a.Dh) *reinterpret_cast<half2_t *>(out) = half2_t{};
        return;
    }
    const int h = head / a.G, r = (row - s.s0) * a.G + head - h * a.G, tile = r / kRows;
    all = wave_sum_f64(all);
    some = wave_sum_f64(some);
    if (too_much(all)) return;
    const Parts in = parts_of(a, s, kRows, h, tile, uniform((int)(unsigned)all), uniform((int)(unsigned)some));
    const int parts = in.count;
    if (parts == 1) return;
    Joined<2> j;
    for (int p0 = first; p0 < parts; p0 += WAVES * kAtOnce) {
        float2 st[kAtOnce];
        float v[kAtOnce][2];
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
            const int64_t at = (int64_t)in.slot(min(p0 + k * WAVES, parts - 1)) * kRows + r - tile * kRows;
            st[k] = *reinterpret_cast<const float2 *>(a.stats + 2 * at);
            const float2 x = *reinterpret_cast<const float2 *>(a.part + at * a.Dh + d);
            v[k][0] = x.x;
            v[k][1] = x.y;
        }
        j.add(st, v, (parts - p0 + WAVES - 1) / WAVES);
    }
    if constexpr (WAVES > 1) {
        __shared__ float o[kWaves][2][64];
        __shared__ float2 ml[kWaves];
        o[wid][0][lane] = j.o[0];
        o[wid][1][lane] = j.o[1];
        ml[wid] = {j.m, j.l};
        __syncthreads();
        if (wid > 0) return;
        float2 st[kWaves];
        float v[kWaves][2];
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            st[w] = ml[w];
            v[w][0] = o[w][0][lane];
            v[w][1] = o[w][1][lane];
        }
        j = Joined<2>();
        j.add(st, v, kWaves);
    }
    const float y = j.l == 0.f ? 0.f : 1.f / j.l;
    if (2 * lane < a.Dh) *reinterpret_cast<half2_t *>(out) = half2_t{f2h(j.o[0] * y), f2h(j.o[1] * y)};
}

// Of the 64 sequences from b0 on those whose numbers do not fit together: named, and the rows that there are of them zeros (of the query
// heads of key head h)
__device__ __forceinline__ void clear_misfits(const AttnArgs &a, int b0, int h)
{
    const int lane = threadIdx.x & 63, b = min(b0 + lane, a.pb.B - 1);
    const bool bad = b0 + lane < a.pb.B && !lane_sequence(a, b0).ok;
    const int from = max(a.pb.starts[b], 0), to = bad ? min(a.pb.starts[b + 1], a.pb.T) : 0;
    if (bad && h == 0 && threadIdx.x < 64) report(a.pb, b);
    for (uint64_t rest = __ballot(from < to); rest; rest &= rest - 1) {
        const int at = __ffsll((unsigned long long)rest) - 1, end = __builtin_amdgcn_readlane(to, at);
        for (int row = __builtin_amdgcn_readlane(from, at) + uniform((int)threadIdx.x >> 6); row < end; row += kWaves)
            for (int d = 4 * lane; d < a.G * a.Dh; d += 256) *reinterpret_cast<half4_t *>(a.out + row * a.ldo + h * a.G * a.Dh + d) = half4_t{};
    }
}

// The same for prompts, and for the few rows of other sequences of the batch: a row to 32 lanes, four columns to a lane, 32 rows of a
// tile and key head to a workgroup (tiles numbered as they are in a batch of any lengths: many find nothing to do).  The last workgroups
// have 64 sequences each to look at: one that does not fit may have more rows than there are tiles numbered for it, or none.
constexpr int kJoinRows = 32;
__global__ void __launch_bounds__(kThreads) paged_attention_join_tiles_kernel(AttnArgs a, Units big, Units few)
{
    constexpr int kRows = 32, kCut = kPrompt / kJoinRows;
    const PagedBatch &pb = a.pb;
    const int lane = threadIdx.x & 63, h = blockIdx.y;
    const int64_t bigs = big.count * kCut;
    const bool prompts = blockIdx.x < bigs;
    if (blockIdx.x >= bigs + few.count) {
        clear_misfits(a, (int)(blockIdx.x - bigs - few.count) * 64, h);
        return;
    }
    const int64_t number = prompts ? blockIdx.x / kCut : blockIdx.x - bigs;
    const int from = prompts ? (int)(blockIdx.x % kCut) * kJoinRows : 0;       // the first row
    // the unit's sequence (as Units::find has it, from what the lanes have of the sequences), all work and that of those before it
    const Units u = {prompts ? big.even : few.even, prompts ? big.per : few.per, prompts ? big.times : few.times, prompts ? big.more : few.more, 0};
    int b = u.even ? (int)(number / u.even) : 0;
    double all = 0., some = 0.;
    Sequence s = {0, 0, 0, false};
    for (int b0 = 0; b0 < pb.B; b0 += 64) {
        const Sequence q = lane_sequence(a, b0);
        const int i = b0 + lane;
        if (!u.even) b += __popcll(__ballot(i < pb.B && u.begin(i + 1, (int)((unsigned)q.s0 + (unsigned)q.n)) <= number));
        const double w = prompts ? big_share_of(a, q).units(a.Hkv) : share_of(a, kRows, q).units;
        all += w;
        some += i < b ? w : 0.;                // (b grows only while all of these are before it)
        if (b >= b0 && b < b0 + 64) s = of_lane(q, b - b0);
    }
    b = uniform(b);
    if (b >= pb.B) return;
    const int tile = uniform((int)(number - u.begin(b, s.s0)));
    const int tile_rows = prompts ? kPrompt : kRows, rows = s.n * a.G, row0 = tile * tile_rows, here = min(tile_rows, rows - row0);
    if (!s.ok || tile < 0 || here <= 0) return;
    auto out_of = [&](int r) { return a.out + (int64_t)(s.s0 + r / a.G) * a.ldo + (h * a.G + r % a.G) * a.Dh; };
    const int d = 4 * (lane & 31), r = from + 2 * (int)(threadIdx.x >> 6) + (lane >> 5), to = min(here, from + kJoinRows);
    if (from >= here) return;
    if (prompts != (rows > a.few)) return;
    all = wave_sum_f64(all);
    some = wave_sum_f64(some);
    if (too_much(all)) return;
    const Parts in = parts_of(a, s, kRows, h, tile, uniform((int)(unsigned)all), uniform((int)(unsigned)some));
    if (in.count == 1) return;
    const float *part = prompts ? a.big_part : a.part, *stats = prompts ? a.big_stats : a.stats;
    constexpr int kAtOnce = 4;                 // parts at once, of two rows
    for (int k = from; k < to; k += 4 * kWaves) {
        Joined<4> j[2];
        for (int p0 = 0; p0 < in.count; p0 += kAtOnce) {
            float2 st[2][kAtOnce];
            float v[2][kAtOnce][4];
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int p = 0; p < kAtOnce; p++) {
                    const int64_t at = (int64_t)in.slot(min(p0 + p, in.count - 1)) * tile_rows + min(r + k - from + 2 * kWaves * e, to - 1);
                    st[e][p] = *reinterpret_cast<const float2 *>(stats + 2 * at);
                    const float4_t x = *reinterpret_cast<const float4_t *>(part + at * a.Dh + min(d, a.Dh - 4));
#pragma unroll
                    for (int i = 0; i < 4; i++) v[e][p][i] = x[i];
                }
#pragma unroll
            for (int e = 0; e < 2; e++) j[e].add(st[e], v[e], in.count - p0);
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float y = j[e].l == 0.f ? 0.f : 1.f / j[e].l;
            const int row = r + k - from + 2 * kWaves * e;
            if (row < to && d < a.Dh)
                *reinterpret_cast<half4_t *>(out_of(row0 + row) + d) = half4_t{f2h(j[e].o[0] * y), f2h(j[e].o[1] * y), f2h(j[e].o[2] * y), f2h(j[e].o[3] * y)};
        }
    }
}

struct Plan {
    int NR, groups, few, big_groups;
    size_t floats(int64_t Dh) const
    {
        return ((size_t)groups * 2 * (16 * NR) + (size_t)big_groups * 2 * kPrompt) * (size_t)(Dh + 2);
    }
};
// Rows of a sequence (tokens by the query heads of a key head) up to which waves of 32 of them read the keys no more often than costs
// less than a prompt's workgroup, where no sequence may have more and where some may: two launches one after the other then.
// (24 sequences of up to 128 rows, as prompts from 64 / 96 / 128 on: 58 / 66 / 39 us, 8 of 192, from 128 / 192: 63 / 92; beside others, 12
// of up to 160, kFew 32 / 64 / 128: 72 / 77 / 92)
constexpr int kNoPrompt = 128, kFew = 32;
Plan plan(int64_t T, int64_t B, int64_t H, int64_t Hkv, int64_t Dh, int64_t max_new, int bytes)
{
    const int64_t G = H / Hkv, rows = (max_new < T ? max_new : T) * G;
    const int NR = rows <= 16 ? 1 : 2;
    if (rows > kNoPrompt) return {2, 2 * device_cus(), B == 1 ? 0 : kFew, 2 * device_cus()};
    return {NR, resident(Dh <= 64 ? 1 : 2, NR, bytes) * device_cus(), INT32_MAX, 0};
}

// Tiles of `rows` rows of the key heads' queries: a tile to as many whole tokens as it holds and one more to a sequence, or, of more
// heads than that, as many to a token as hold it (more than it takes where one does not divide the other)
Units tiles_of(const AttnArgs &a, int rows)
{
    const int64_t most = ((int64_t)a.max_new * a.G + rows - 1) / rows;
    return a.G > rows ? make_units(a.pb.T, a.pb.B, 1, (a.G + rows - 1) / rows, 0, most) : make_units(a.pb.T, a.pb.B, rows / a.G, 1, 1, most);
}
int launch_join_prompts(const AttnArgs &a, hipStream_t st)
{
    const Units few = a.few ? tiles_of(a, 32) : Units{1, 1, 1, 1, 0}, big = tiles_of(a, kPrompt);
    const int64_t grid = few.count + big.count * (kPrompt / kJoinRows) + (a.pb.B + 63) / 64;
    hipLaunchKernelGGL(paged_attention_join_tiles_kernel, dim3((unsigned)grid, (unsigned)a.Hkv), dim3(kThreads), 0, st, a, big, few);
    return launch_status("paged_attention (parts)");
}
template <int NR>
int launch_join(const AttnArgs &a, hipStream_t st)
{
    if (a.big_groups) return launch_join_prompts(a, st);
    const int64_t rh = (int64_t)a.pb.T * a.H;
    if (rh < 4 * device_cus()) hipLaunchKernelGGL((paged_attention_join_kernel<NR, kWaves>), dim3((unsigned)rh + 1), dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((paged_attention_join_kernel<NR, 1>), dim3((unsigned)((rh + kWaves - 1) / kWaves) + 1), dim3(kThreads), 0, st, a);
    return launch_status("paged_attention (parts)");
}
template <int ND, int NR, class P>
int launch(const AttnArgs &a, hipStream_t st)
{
    hipLaunchKernelGGL((paged_attention_kernel<ND, NR, P>), dim3((unsigned)a.groups), dim3(kThreads), 0, st, a);
    const int rc = launch_status("paged_attention");
    return rc ? rc : launch_join<NR>(a, st);
}
template <int ND, class P>
int launch_prompts(const AttnArgs &a, hipStream_t st)
{
    hipLaunchKernelGGL((paged_prompt_kernel<ND, P>), dim3((unsigned)a.big_groups), dim3(kBigThreads), 0, st, a);
    const int rc = launch_status("paged_attention (prompts)");
    if (rc) return rc;
    return a.few > 0 ? launch<ND, 2, P>(a, st) : launch_join_prompts(a, st);        // (one sequence: there are no others)
}
template <class P>
int launch(const AttnArgs &a, int NR, hipStream_t st)
{
    if (a.big_groups) return a.Dh <= 64 ? launch_prompts<1, P>(a, st) : launch_prompts<2, P>(a, st);
    if (a.Dh <= 64) return NR == 1 ? launch<1, 1, P>(a, st) : launch<1, 2, P>(a, st);
    return NR == 1 ? launch<2, 1, P>(a, st) : launch<2, 2, P>(a, st);
}

}  // namespace

CACTI_API size_t cacti_hip_paged_attention_workspace(int64_t T, int64_t B, int64_t H, int64_t Hkv, int64_t Dh, int64_t max_new)
{
    if (T <= 0 || B <= 0 || H <= 0 || Hkv <= 0 || Dh <= 0 || max_new <= 0 || H % Hkv) return 0;
    const Plan p = plan(T, B, H, Hkv, Dh, max_new, 1);        // (of 16 bits: no more)
    return p.floats(Dh) * 4;
}

CACTI_API int cacti_hip_paged_attention_f16(int64_t T, int64_t B, int64_t H, int64_t Hkv, int64_t Dh, int64_t max_new, float alpha,
                                            const void *q, int64_t ldq, const void *k_pages, const void *v_pages, const void *k_scale,
                                            const void *v_scale, int bits, int64_t P, int64_t page, const void *table, int64_t ldt, int64_t W,
                                            const void *starts, const void *lens, void *out, int64_t ldo, void *workspace,
                                            size_t workspace_bytes, void *status, void *stream)
{
    PagedBatch pb;
    const int rc = paged_batch("paged_attention", T, B, H, Hkv, Dh, max_new, table, ldt, W, starts, lens, status, k_pages, v_pages, k_scale,
                               v_scale, bits, P, page, &pb);
    if (rc) return rc;
    CACTI_REQUIRE(q && out, CACTI_E_INVALID, "paged_attention: null pointer");
    CACTI_REQUIRE(ldq >= H * Dh && ldo >= H * Dh && ldq % 4 == 0 && ldo % 4 == 0 && aligned(q, 8) && aligned(out, 8), CACTI_E_INVALID,
                  "paged_attention: operands must be 8-byte aligned with row pitches that are multiples of 4 and hold a row");
    CACTI_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= cacti_hip_paged_attention_workspace(T, B, H, Hkv, Dh, max_new),
                  CACTI_E_INVALID, "paged_attention: workspace too small or not 16-byte aligned");
    CACTI_REQUIRE(fabsf(alpha) < INFINITY, CACTI_E_INVALID, "paged_attention: alpha is not finite");
    // tiles of 16 rows of one sequence, of all, whichever is less; work is counted in 32 bits
    const int64_t most = (max_new < T ? max_new : T) * (H / Hkv) / 16 + 1, tiles = T * (H / Hkv) / 16 + B < most * B ? T * (H / Hkv) / 16 + B : most * B;
    CACTI_REQUIRE(T * H < (1 << 24) && tiles * Hkv < INT32_MAX / (W * page / kStep + 1 + begin_of(32)), CACTI_E_NOTIMPL,
                  "paged_attention: too many rows and positions in one call");
    CACTI_REQUIRE(!rows_share(T, q, ldq, H * Dh, out, ldo, H * Dh), CACTI_E_INVALID,
                  "paged_attention: the output shares memory with the queries, which other workgroups read");
    const Plan p = plan(T, B, H, Hkv, Dh, max_new, bits / 8);
    float *part = (float *)workspace;
    const size_t small = (size_t)p.groups * 2 * (16 * p.NR);
    const AttnArgs a = {pb, (int)H, (int)Hkv, (int)(H / Hkv), (int)Dh, padded_dim((int)Dh), (int)(max_new < T ? max_new : T), p.groups,
                        magic_of(page), fabsf(alpha), alpha < 0.f ? 0x80008000u : 0u, (const half_t *)q, ldq, k_pages, v_pages, (const float *)k_scale,
                        (const float *)v_scale, (half_t *)out, ldo, part, part + small * Dh, p.few, p.big_groups,
                        part + small * (Dh + 2), part + small * (Dh + 2) + (size_t)p.big_groups * 2 * kPrompt * Dh};
    return bits == 8 ? launch<uint8_t>(a, p.NR, (hipStream_t)stream) : launch<half_t>(a, p.NR, (hipStream_t)stream);
}
