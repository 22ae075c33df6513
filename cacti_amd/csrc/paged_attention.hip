// Causal attention of the new rows of a ragged batch over a paged cache, in e4m3 with a scale per page and head or in f16:
//   o = sum_j softmax_j(alpha q . k_j) v_j     over the positions j up to the row's own
//
// One pass over the keys with a running maximum.  The codes meet the queries as they are (e4m3 to f16 is exact) and a page's
// scales join the scores: with t_j = alpha ks q . k_j log2 e + log2 vs and m the maximum of t so far,
//   w_j = 2^(t_j - m) <= 1,  o = sum w_j code(v_j) / sum w_j / vs
// so that the weight that meets a code already holds its page's scale, and no w exceeds f16 whatever the scales are.
// Scores, maxima, sums and o are fp32; w is rounded to f16 for the matrix instruction (2^-11 relative, each on its own, which
// is what the rounding of the output adds once more).
//
// A workgroup has 16 NR rows (tokens of a sequence by the query heads that share a key head), a key head and a part of the
// positions; its four waves take 32 positions in turn and put their sums together at the end.  The products are formed
// transposed, S^T = K Q^T and O^T = V^T W^T with v_mfma_f32_16x16x32_f16: a lane then holds the scores of one row, at keys
// that are exactly those its part of the second product's operand wants, so that w never leaves the lane.  Keys come from
// memory in the order the instruction takes them (16 columns of a key to a lane); V, whose operand is a column of eight
// keys, is read as rows of 8 columns and turned with byte permutes.  No LDS, no barrier inside.
#include "paged.h"

using namespace cacti;

namespace {

constexpr int kThreads = 256, kWaves = 4, kStep = 32;
constexpr int kEntries = 128;                  // pages of a workgroup's positions at a time
constexpr int kSegment = 2048;                 // positions of them: 128 pages of 16

struct AttnArgs {
    PagedBatch pb;
    Units units;
    int H, Hkv, G, Dh, Dp, max_new;
    int chunk, splits;                         // positions of a workgroup, workgroups behind one another along a sequence
    float alpha;
    const half_t *q;
    int64_t ldq;
    const void *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    half_t *out;
    int64_t ldo;
    float *part, *stats;                       // [split][T][H][Dh], [split][T][H][2]
};

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
    __device__ __forceinline__ half8_t part(int s) const
    {
        Frag f;
        f.u[0] = cvt8(w[2 * s], false);
        f.u[1] = cvt8(w[2 * s], true);
        f.u[2] = cvt8(w[2 * s + 1], false);
        f.u[3] = cvt8(w[2 * s + 1], true);
        return f.h;
    }
};
template <>
struct KPiece<half_t> {
    half8_t w[2];
    __device__ __forceinline__ void load(const half_t *p)
    {
        w[0] = *reinterpret_cast<const half8_t *>(p);
        w[1] = *reinterpret_cast<const half8_t *>(p + 8);
    }
    __device__ __forceinline__ half8_t part(int s) const { return w[s]; }
    __device__ __forceinline__ void zero() { w[0] = w[1] = half8_t{}; }
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
    __device__ __forceinline__ bool odd(int i) const       // a NaN among them
    {
        bool any = false;
#pragma unroll
        for (int j = 0; j < VD / 4; j++) {
            const unsigned x = w[i][j] & 0x7f7f7f7fu;
            any = any || ((x + 0x01010101u) & 0x80808080u);
        }
        return any;
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
    __device__ __forceinline__ bool odd(int i) const       // a NaN or an infinity among them
    {
        bool any = false;
#pragma unroll
        for (int j = 0; j < VD / 2; j++) any = any || (w[i][j] & 0x7c00u) == 0x7c00u || (w[i][j] & 0x7c000000u) == 0x7c000000u;
        return any;
    }
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

__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// What a page of a workgroup's positions is: where its rows of this head begin and what its scales make of a score
struct Entry {
    int64_t at;
    float c, lg, iv;                           // alpha ks log2 e, log2 vs, 1 / vs
};

// ND: pieces of 64 columns of a head
template <int ND, int NR, class P>
__global__ void __launch_bounds__(kThreads) paged_attention_kernel(AttnArgs a)
{
    constexpr int VD = 4 * ND;                 // columns of V of a lane
    constexpr int NS = 2 * ND;                 // matrix instructions along the columns of a key
    __shared__ Entry entry[kEntries];
    __shared__ float merged[kWaves][16 * NR][VD * 16 + 4];
    __shared__ float wave_m[kWaves][16 * NR], wave_l[kWaves][16 * NR];
    const PagedBatch &pb = a.pb;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
    const int64_t x = blockIdx.x / a.splits;
    const int split = (int)(blockIdx.x - x * a.splits), h = blockIdx.y;
    int tile;
    const int b = a.units.find(pb, x, &tile);
    if (b >= pb.B) return;
    const Sequence s = sequence(pb, b, (int64_t)pb.W * pb.page, a.max_new);
    const int rows = s.n * a.G, row0 = tile * 16 * NR;
    if (s.s0 < 0 || s.n < 0 || s.s0 > pb.T - s.n || row0 < 0 || row0 >= rows) return;
    if (!s.ok) {                               // rows that there are at positions that there are not: zeros
        if (threadIdx.x == 0) report(pb, b);
        if (split == 0)
            for (int i = threadIdx.x; i < 16 * NR * a.Dh; i += kThreads) {
                const int r = row0 + i / a.Dh, d = i % a.Dh;
                if (r < rows) a.out[(int64_t)(s.s0 + r / a.G) * a.ldo + (h * a.G + r % a.G) * a.Dh + d] = (half_t)0.f;
            }
        return;
    }
    const int end = s.first + min(rows - 1, row0 + 16 * NR - 1) / a.G + 1;         // positions that some row of the tile sees
    const int c0 = split * a.chunk, c1 = min(end, c0 + a.chunk);
    if (c0 >= c1) return;

    // the lane's row of each 16: its query, its last position
    half8_t q[NR][NS];
    int last[NR];
    float m[NR], l[NR];
    float4_t o[NR][VD];
    int least = INT32_MAX;                     // positions up to here are seen by every row
#pragma unroll
    for (int n = 0; n < NR; n++) {
        const int r = min(row0 + 16 * n + r16, rows - 1), t = r / a.G;
        last[n] = s.first + t;
        const half_t *qr = a.q + (int64_t)(s.s0 + t) * a.ldq + (h * a.G + r - t * a.G) * a.Dh;
#pragma unroll
        for (int c = 0; c < ND; c++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                Frag f;
#pragma unroll
                for (int j = 0; j < 2; j++) {  // pieces of four columns: Dh is a multiple of 4
                    const int d = 64 * c + 16 * g + 8 * k + 4 * j;
                    const u2_t w = *reinterpret_cast<const u2_t *>(qr + min(d, a.Dh - 4));
                    f.u[2 * j] = d < a.Dh ? w[0] : 0u;
                    f.u[2 * j + 1] = d < a.Dh ? w[1] : 0u;
                }
                q[n][2 * c + k] = f.h;
            }
        m[n] = -INFINITY;
        l[n] = 0.f;
#pragma unroll
        for (int i = 0; i < VD; i++) o[n][i] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    least = s.first + row0 / a.G;

    const P *kp = (const P *)a.k_pages, *vp = (const P *)a.v_pages;
    const float log2e = 1.44269504088896340736f;
    for (int seg = c0; seg < c1; seg += kSegment) {
        const int seg1 = min(c1, seg + kSegment), p0 = seg / pb.page, np = (seg1 - 1) / pb.page - p0 + 1;
        if (seg > c0) __syncthreads();
        for (int i = threadIdx.x; i < np; i += kThreads) {
            int id = pb.table[(int64_t)b * pb.ldt + p0 + i];
            if (id < 0 || id >= pb.P) {
                report(pb, b);
                id = 0;                        // its rows are unspecified, not its reads
            }
            const int64_t ph = (int64_t)id * a.Hkv + h;
            Entry e = {ph * pb.page * a.Dp, a.alpha * log2e, 0.f, 1.f};
            if (sizeof(P) == 1) {
                e.c *= a.k_scale[ph];
                e.lg = log2f(a.v_scale[ph]);
                e.iv = 1.f / a.v_scale[ph];
            }
            entry[i] = e;
        }
        __syncthreads();
        for (int j0 = seg + kStep * wid; j0 < seg1; j0 += kStep * kWaves) {
            KPiece<P> kk[2][ND];
            VBlock<P, VD> vv;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int j = min(j0 + 8 * (r16 >> 2) + 4 * t + (r16 & 3), seg1 - 1), pg = j / pb.page;
                const P *row = kp + entry[pg - p0].at + (j - pg * pb.page) * a.Dp;
#pragma unroll
                for (int c = 0; c < ND; c++) {
                    kk[t][c].load(row + min(64 * c + 16 * g, a.Dp - 16));
                    // (there the query is zero, and an infinity of another column would make a NaN with it)
                    if constexpr (sizeof(P) == 2)
                        if (64 * c + 16 * g >= a.Dp) kk[t][c].zero();
                }
            }
            const int mine = min(j0 + 8 * g, seg1 - 1) / pb.page - p0;       // page of the lane's eight keys
            const float ec = entry[mine].c, lg = entry[mine].lg, iv = entry[mine].iv;
            const P *vrow = vp + entry[mine].at + min(VD * r16, a.Dp - VD);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int j = min(j0 + 8 * g + i, seg1 - 1);
                vv.load(i, vrow + (j - (mine + p0) * pb.page) * a.Dp);
            }
            float4_t sc[NR][2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
#pragma unroll
                for (int n = 0; n < NR; n++) sc[n][t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NS; c++) {
                    const half8_t kf = kk[t][c / 2].part(c & 1);
#pragma unroll
                    for (int n = 0; n < NR; n++) sc[n][t] = mfma(kf, q[n][c], sc[n][t]);
                }
            }
            const bool edge = j0 + kStep - 1 > min(least, seg1 - 1);       // (the same in every lane)
            half8_t w[NR];
#pragma unroll
            for (int n = 0; n < NR; n++) {
                float t[8], mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float raw = i < 4 ? sc[n][0][i & 3] : sc[n][1][i & 3];
                    t[i] = __builtin_fmaf(raw, ec, lg);
                    if (edge && j0 + 8 * g + i > min(last[n], seg1 - 1)) t[i] = -INFINITY;
                    mx = fmaxf(mx, t[i]);
                }
                mx = with32(with16(mx, OpMax()), OpMax());
                const float mn = fmaxf(m[n], mx), base = finite_max(mn);
                const float f = exp2_of(m[n] - base);
                m[n] = mn;
                float sum = 0.f;
                Frag p;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    t[i] = exp2_of(t[i] - base);
                    sum += t[i];
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const half2_t pair = {f2h(t[2 * i]), f2h(t[2 * i + 1])};
                    p.u[i] = __builtin_bit_cast(unsigned, pair);
                }
                l[n] = l[n] * f + sum * iv;
                w[n] = p.h;
#pragma unroll
                for (int i = 0; i < VD; i++) o[n][i] *= f;
            }
            bool odd = false;
            if (edge) {
                // what no row of the tile sees is nothing; a NaN or an infinity that some rows see must not meet the zero
                // weights of the others
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int j = j0 + 8 * g + i;
                    if (j >= seg1) vv.zero(i);
                    else odd = odd || (j > least && vv.odd(i));
                }
                odd = __ballot(odd) != 0;
            }
            if (!odd) {
#pragma unroll
                for (int c = 0; c < VD / 2; c++) {
                    half8_t v0, v1;
                    vv.columns(c, &v0, &v1);
#pragma unroll
                    for (int n = 0; n < NR; n++) {
                        o[n][2 * c] = mfma(v0, w[n], o[n][2 * c]);
                        o[n][2 * c + 1] = mfma(v1, w[n], o[n][2 * c + 1]);
                    }
                }
            } else {
                for (int j = j0; j < min(j0 + kStep, seg1); j++) {          // one key at a time, to the rows that see it
                    VBlock<P, VD> one = vv;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (j0 + 8 * g + i != j) one.zero(i);
#pragma unroll
                    for (int c = 0; c < VD / 2; c++) {
                        half8_t v0, v1;
                        one.columns(c, &v0, &v1);
#pragma unroll
                        for (int n = 0; n < NR; n++) {
                            const float4_t z = {0.f, 0.f, 0.f, 0.f};
                            const float4_t a0 = mfma(v0, w[n], z), a1 = mfma(v1, w[n], z);
                            if (j <= last[n]) {
                                o[n][2 * c] += a0;
                                o[n][2 * c + 1] += a1;
                            }
                        }
                    }
                }
            }
        }
    }

    // the four waves' sums: a lane has columns VD (4 g + i) + c of its row in o[.][c][i]
#pragma unroll
    for (int n = 0; n < NR; n++) {
        l[n] = with32(with16(l[n], OpSum()), OpSum());
        if (g == 0) {
            wave_m[wid][16 * n + r16] = m[n];
            wave_l[wid][16 * n + r16] = l[n];
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int c = 0; c < VD; c++) merged[wid][16 * n + r16][VD * (4 * g + i) + c] = o[n][c][i];
    }
    __syncthreads();
    const bool whole = s.first + s.n <= a.chunk;             // the sequence has one part: no partial sums
    for (int i = threadIdx.x; i < 16 * NR * (a.Dh / 4); i += kThreads) {
        const int r = i / (a.Dh / 4), d = 4 * (i - r * (a.Dh / 4));
        if (row0 + r >= rows) break;
        float mx = wave_m[0][r];
#pragma unroll
        for (int w = 1; w < kWaves; w++) mx = fmaxf(mx, wave_m[w][r]);
        const float base = finite_max(mx);
        float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float f = exp2_of(wave_m[w][r] - base);
            sum += f * wave_l[w][r];
#pragma unroll
            for (int k = 0; k < 4; k++) acc[k] += f * merged[w][r][d + k];
        }
        const int t = (row0 + r) / a.G, head = h * a.G + row0 + r - t * a.G;
        if (whole) {
            const float y = sum == 0.f ? 0.f : 1.f / sum;
            half4_t v;
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = f2h(acc[k] * y);
            *reinterpret_cast<half4_t *>(a.out + (int64_t)(s.s0 + t) * a.ldo + head * a.Dh + d) = v;
        } else {
            const int64_t at = ((int64_t)split * pb.T + s.s0 + t) * a.H + head;
            *reinterpret_cast<float4_t *>(a.part + at * a.Dh + d) = float4_t{acc[0], acc[1], acc[2], acc[3]};
            if (d == 0) {
                a.stats[2 * at] = mx;
                a.stats[2 * at + 1] = sum;
            }
        }
    }
}

// The parts of a row put together: a wave per row and head, two columns per lane.
__global__ void __launch_bounds__(kThreads) paged_attention_join_kernel(AttnArgs a)
{
    const PagedBatch &pb = a.pb;
    const int lane = threadIdx.x & 63;
    const int64_t rh = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    const int row = (int)(rh / a.H), head = (int)(rh - (int64_t)row * a.H);
    if (row >= pb.T) return;
    const int b = count_below(pb.B, row, [&](int i) { return pb.starts[i]; });
    if (b >= pb.B) return;
    const Sequence s = sequence(pb, b, (int64_t)pb.W * pb.page, a.max_new);
    if (!s.ok || row < s.s0 || row >= s.s0 + s.n || s.first + s.n <= a.chunk) return;
    const int parts = (s.first + row - s.s0) / a.chunk + 1;
    const int64_t step = (int64_t)pb.T * a.H;
    float mx = -INFINITY;
    for (int p = lane; p < parts; p += 64) mx = fmaxf(mx, a.stats[2 * (p * step + rh)]);
    const float base = finite_max(wave_max(mx));
    const int d = min(2 * lane, a.Dh - 2);
    float sum = 0.f, o0 = 0.f, o1 = 0.f;
    for (int p = 0; p < parts; p++) {
        const int64_t at = p * step + rh;
        const float f = exp2_of(a.stats[2 * at] - base);
        const float2 v = *reinterpret_cast<const float2 *>(a.part + at * a.Dh + d);
        sum += f * a.stats[2 * at + 1];
        o0 += f * v.x;
        o1 += f * v.y;
    }
    const float y = sum == 0.f ? 0.f : 1.f / sum;
    if (2 * lane < a.Dh) {
        const half2_t v = {f2h(o0 * y), f2h(o1 * y)};
        *reinterpret_cast<half2_t *>(a.out + row * a.ldo + head * a.Dh + d) = v;
    }
}

struct Plan {
    int NR, chunk, splits;
    Units units;
};

Plan plan(int64_t T, int64_t B, int64_t H, int64_t Hkv, int64_t max_new, int64_t longest)
{
    const int64_t G = H / Hkv;
    Plan p;
    if (max_new > T) max_new = T;
    p.NR = max_new * G <= 16 ? 1 : 2;
    const int64_t tile = 16 * p.NR;
    // (s1 G) / tile - (s0 G) / tile + 1 tiles are numbered from starts / (tile / G) + b on where G divides the tile; otherwise
    // a tile is taken to hold no more tokens than fit whole
    const int64_t tokens = G >= tile ? 1 : tile / G;
    const int64_t most = (max_new * G + tile - 1) / tile;
    p.units = G >= tile ? Units{(int)most, 1, 1, most * B} : make_units(T, B, tokens, 1, most);
    const int64_t want = 4 * device_cus(), have = p.units.count * Hkv;
    int64_t splits = want / have;
    const int64_t limit = (longest + 127) / 128;
    if (splits > limit) splits = limit;
    if (splits < 1) splits = 1;
    p.chunk = (int)((longest + splits - 1) / splits + 127) / 128 * 128;
    p.splits = (int)((longest + p.chunk - 1) / p.chunk);
    return p;
}

template <class P>
int launch(const AttnArgs &a, const Plan &p, hipStream_t st)
{
    const dim3 grid((unsigned)(p.units.count * p.splits), (unsigned)a.Hkv), block(kThreads);
    if (a.Dh <= 64) {
        if (p.NR == 1) hipLaunchKernelGGL((paged_attention_kernel<1, 1, P>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((paged_attention_kernel<1, 2, P>), grid, block, 0, st, a);
    } else {
        if (p.NR == 1) hipLaunchKernelGGL((paged_attention_kernel<2, 1, P>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((paged_attention_kernel<2, 2, P>), grid, block, 0, st, a);
    }
    const int rc = launch_status("paged_attention");
    if (rc || p.splits == 1) return rc;
    const int64_t waves = (int64_t)a.pb.T * a.H;
    hipLaunchKernelGGL(paged_attention_join_kernel, dim3((unsigned)((waves + kWaves - 1) / kWaves)), block, 0, st, a);
    return launch_status("paged_attention (parts)");
}

}  // namespace

CACTI_API size_t cacti_hip_paged_attention_workspace(int64_t T, int64_t B, int64_t H, int64_t Hkv, int64_t Dh, int64_t max_new, int64_t page,
                                                     int64_t W)
{
    if (T <= 0 || B <= 0 || H <= 0 || Hkv <= 0 || Dh <= 0 || max_new <= 0 || page <= 0 || W <= 0 || H % Hkv) return 0;
    const Plan p = plan(T, B, H, Hkv, max_new, W * page);
    return p.splits == 1 ? 0 : (size_t)p.splits * (size_t)(T * H) * (size_t)(Dh + 2) * 4;
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
    const Plan p = plan(T, B, H, Hkv, max_new, W * page);
    const size_t need = cacti_hip_paged_attention_workspace(T, B, H, Hkv, Dh, max_new, page, W);
    CACTI_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need), CACTI_E_INVALID,
                  "paged_attention: workspace too small or not 16-byte aligned");
    CACTI_REQUIRE(p.units.count * p.splits < (1 << 24) && (T * H + kWaves - 1) / kWaves < (1 << 24), CACTI_E_NOTIMPL,
                  "paged_attention: too many rows in one call");
    float *part = (float *)workspace;
    const AttnArgs a = {pb, p.units, (int)H, (int)Hkv, (int)(H / Hkv), (int)Dh, padded_dim((int)Dh), (int)(max_new < T ? max_new : T), p.chunk,
                        p.splits, alpha, (const half_t *)q, ldq, k_pages, v_pages, (const float *)k_scale, (const float *)v_scale,
                        (half_t *)out, ldo, part, part ? part + (size_t)p.splits * T * H * Dh : nullptr};
    return bits == 8 ? launch<uint8_t>(a, p, (hipStream_t)stream) : launch<half_t>(a, p, (hipStream_t)stream);
}
