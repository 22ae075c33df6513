// New keys and values into the pages of a cache, rotated on the way, with the queries of the same rows.
//
//   k'[d] = k[d] cos[p][d] - k[d + Dh/2] sin[p][d]   (d < Dh/2; the other half: k[d] cos[p][d] + k[d - Dh/2] sin[p][d])
// with the products exact (22 of 24 bits) and one rounding of their sum in fp32, then one into the page: to f16, or to e4m3
// of k' / scale with the scale 2^e of the page and head.  A power of two costs the quotient no rounding and e4m3 nothing of
// its precision (it has an exponent of its own), and codes that are there already can be carried over to a larger scale
// exactly, but for those that become subnormal.
//
// A workgroup owns a page and a head: it holds the new rows of that page in registers, takes the least scale that holds them and
// no less than that of older rows, codes those again where it grew, and writes.  No other workgroup touches that page and head.
// Bound by memory: four sequences of up to 2048 rows, 32 heads of 100 in 8 bits 38 to 40 us, of which 18 are the queries' (reading the
// rows once for the scale and again for the codes, two columns at a time: 56.4), in 16 bits 53; 96 of up to 6 rows, 8 heads of 128: 5.4 us;
// one row 4.2 us, latency.
#include "operands.h"
#include "paged.h"

using namespace cacti;

namespace cacti {

int paged_batch(const char *who, int64_t T, int64_t B, int64_t H, int64_t Hkv, int64_t Dh, int64_t max_new, const void *table,
                int64_t ldt, int64_t W, const void *starts, const void *lens, void *status, const void *k_pages, const void *v_pages,
                const void *k_scale, const void *v_scale, int bits, int64_t P, int64_t page, PagedBatch *pb)
{
    CACTI_REQUIRE(T > 0 && B > 0 && H > 0 && Hkv > 0 && P > 0 && W > 0 && max_new > 0, CACTI_E_INVALID, "%s: empty shape", who);
    CACTI_REQUIRE(table && starts && lens && k_pages && v_pages, CACTI_E_INVALID, "%s: null pointer", who);
    CACTI_REQUIRE(bits == 8 || bits == 16, CACTI_E_INVALID, "%s: pages of 8 or 16 bits", who);
    CACTI_REQUIRE((bits == 8) == (k_scale && v_scale) && (bits == 8 || (!k_scale && !v_scale)), CACTI_E_INVALID,
                  "%s: pages of 8 bits have scales, pages of 16 bits none", who);
    CACTI_REQUIRE(H % Hkv == 0, CACTI_E_INVALID, "%s: %lld query heads for %lld key heads", who, (long long)H, (long long)Hkv);
    CACTI_REQUIRE(Dh % 4 == 0 && Dh >= 4 && Dh <= 128, CACTI_E_NOTIMPL, "%s: need Dh %% 4 == 0 and Dh <= 128", who);
    CACTI_REQUIRE(page % 16 == 0 && page >= 16 && page <= 256, CACTI_E_NOTIMPL, "%s: pages of 16 to 256 positions, a multiple of 16", who);
    CACTI_REQUIRE(T <= INT32_MAX / H && B < 65536 * 16 && P <= INT32_MAX && W <= (1 << 30) / page && H <= 4096 && ldt >= W, CACTI_E_NOTIMPL,
                  "%s: too many rows, sequences or pages, or a table pitch below its width", who);
    CACTI_REQUIRE(aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(table, 4) && aligned(starts, 4) && aligned(lens, 4) &&
                      aligned(k_scale, 4) && aligned(v_scale, 4) && aligned(status, 4),
                  CACTI_E_INVALID, "%s: pages must be 16-byte aligned", who);
    *pb = {(int)T, (int)B, (int)page, (int)W, ldt, (int)P, (const int *)starts, (const int *)lens, (const int *)table, (int *)status};
    return 0;
}

}  // namespace cacti

namespace {

constexpr int kMinExp = -32, kMaxExp = 15;     // of a page's scale: 2^-24 / 448 and beyond sqrt(2) 65504 / 448

struct AppendArgs {
    PagedBatch pb;
    Units units;
    int H, Hkv, Dh, max_new;
    int per, slices;                           // items of a row of a head; workgroups of a row of the queries
    unsigned per_magic;                        // x / per = x * per_magic >> 16 for items x of a page
    int64_t n_pos;                             // rows of cos, sin
    const half_t *q, *k, *v, *cos, *sin;
    int64_t ldq, ldk, ldv, ldqo;
    half_t *q_out;
    void *k_pages, *v_pages;
    float *k_scale, *v_scale;
};

// HV columns of the left half of a head and their partners in the right half.  HV columns to an item, the last one of a row
// reaching back to have as many (what it shares with the one before it both write alike), at any even column.
template <int HV>
struct Loaded {
    typedef half_t vec_t __attribute__((ext_vector_type(HV)));
    typedef vec_t any_t __attribute__((aligned(4)));
    vec_t l, r;
    __device__ __forceinline__ void load(const half_t *x, int half)
    {
        l = *reinterpret_cast<const any_t *>(x);
        r = *reinterpret_cast<const any_t *>(x + half);
    }
};
template <int HV>
struct Item {
    float a[HV], b[HV];
    __device__ __forceinline__ void plain(const Loaded<HV> &x)
    {
#pragma unroll
        for (int i = 0; i < HV; i++) {
            a[i] = h2f(x.l[i]);
            b[i] = h2f(x.r[i]);
        }
    }
    __device__ __forceinline__ void rotated(const Loaded<HV> &x, const Loaded<HV> &c, const Loaded<HV> &s)
    {
#pragma unroll
        for (int i = 0; i < HV; i++) {
            a[i] = h2f(x.l[i]) * h2f(c.l[i]) - h2f(x.r[i]) * h2f(s.l[i]);
            b[i] = h2f(x.r[i]) * h2f(c.r[i]) + h2f(x.l[i]) * h2f(s.r[i]);
        }
    }
    __device__ __forceinline__ float amax() const          // of the finite ones
    {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < HV; i++) {
            const float x = fabsf(a[i]), y = fabsf(b[i]);
            m = fmaxf(m, x < INFINITY ? x : 0.f);
            m = fmaxf(m, y < INFINITY ? y : 0.f);
        }
        return m;
    }
};

template <int HV>
__device__ __forceinline__ void put(half_t *to, const float (&x)[HV], float)
{
    typename Loaded<HV>::vec_t h;
#pragma unroll
    for (int i = 0; i < HV; i++) h[i] = f2h(x[i]);
    *reinterpret_cast<typename Loaded<HV>::any_t *>(to) = h;
}
// e4m3, to nearest, ties to even; NaN and infinities become NaN
template <int HV>
__device__ __forceinline__ void put(uint8_t *to, const float (&x)[HV], float inv)
{
    if constexpr (HV == 8) {
        typedef unsigned two_t __attribute__((ext_vector_type(2)));
        typedef two_t any_t __attribute__((aligned(2)));
        two_t w;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
            w[i] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, lo, true);
        }
        *reinterpret_cast<any_t *>(to) = w;
    } else
        *reinterpret_cast<uint16_t *>(to) = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
}

// the least 2^e >= amax / 448 with e in range
__device__ __forceinline__ float scale_for(float amax)
{
    int e = kMinExp;
    if (amax > 0.f) {
        int x;
        const float m = frexpf(amax, &x);                  // amax = m 2^x, 1/2 <= m < 1; 448 = 0.875 2^9
        e = m > 0.875f ? x - 8 : x - 9;
        e = min(max(e, kMinExp), kMaxExp);
    }
    return ldexpf(1.f, e);
}

// The page's scale for new values up to mx and, if there are older positions, what was; their codes, coded again if it grew
template <int T>
__device__ __forceinline__ float rescale(uint8_t *page, int slot0, int Dp, float mx, float was)
{
    const float to = scale_for(mx);
    if (slot0 == 0) return to;
    if (was >= to) return was;
    const float f = was / to;
    for (int i = threadIdx.x; i < slot0 * (Dp / 16); i += T) {
        int4 w = reinterpret_cast<int4 *>(page)[i];
        int *x = reinterpret_cast<int *>(&w);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float c0 = __builtin_amdgcn_cvt_f32_fp8(x[k], 0), c1 = __builtin_amdgcn_cvt_f32_fp8(x[k], 1);
            const float c2 = __builtin_amdgcn_cvt_f32_fp8(x[k], 2), c3 = __builtin_amdgcn_cvt_f32_fp8(x[k], 3);
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c0 * f, c1 * f, 0, false);
            x[k] = __builtin_amdgcn_cvt_pk_fp8_f32(c2 * f, c3 * f, lo, true);
        }
        reinterpret_cast<int4 *>(page)[i] = w;
    }
    return to;
}

// Workgroups of T threads: one for each unit (page of a sequence) and head, whose rows they hold, two items of the keys and of the
// values to a thread; then those that name 64 sequences each that do not fit together (units are numbered by starts that do not fall, and
// a sequence behind which they do may have none); then groups of up to 256 threads, `slices` of them for kRows rows of the queries.
// Rows of the queries to a thread (4 sequences of up to 2048 rows, 32 heads of 100: 1 / 2 / 4 rows 38.5 / 37.3 / 37.9 us)
template <int T>
constexpr int rows_of() { return T == 64 ? 1 : 2; }

template <int T, int HV, class P>
__global__ void __launch_bounds__(T) paged_append_kernel(AppendArgs a)
{
    constexpr int kRows = rows_of<T>();
    const PagedBatch &pb = a.pb;
    const int64_t limit = min((int64_t)pb.W * pb.page, a.n_pos);
    const int pages = (int)a.units.count * a.Hkv, named = pages + (pb.B + 63) / 64, half = a.Dh / 2;
    auto column = [&](int i) { return min(i * HV, half - HV); };
    if ((int)blockIdx.x >= named) {
        constexpr int TQ = T < 256 ? T : 256;
        const int u = ((int)blockIdx.x - named) * (T / TQ) + __builtin_amdgcn_readfirstlane((int)threadIdx.x / TQ), r = u / a.slices;
        const int i = (u - r * a.slices) * TQ + (int)threadIdx.x % TQ, h = min(i / a.per, a.H - 1), d = column(i - i / a.per * a.per), row0 = r * kRows;
        if (row0 >= pb.T) return;
        Loaded<HV> x[kRows];                   // (these rows there are, if not of a sequence)
#pragma unroll
        for (int e = 0; e < kRows; e++) x[e].load(a.q + (int64_t)min(row0 + e, pb.T - 1) * a.ldq + h * a.Dh + d, half);
        Sequence of[kRows];
#pragma unroll
        for (int e = 0; e < kRows; e++) of[e].ok = false;
        for (int b0 = 0; b0 < pb.B; b0 += 64) {
            const Sequence s = lane_sequence(pb, b0, limit, a.max_new);
#pragma unroll
            for (int e = 0; e < kRows; e++) {
                const uint64_t hit = __ballot(s.ok && row0 + e >= s.s0 && row0 + e - s.s0 < s.n);
                if (hit) of[e] = of_lane(s, __ffsll((unsigned long long)hit) - 1);
            }
        }
        Loaded<HV> c[kRows], sn[kRows];
#pragma unroll
        for (int e = 0; e < kRows; e++) {
            const int64_t pos = of[e].ok ? of[e].first + row0 + e - of[e].s0 : 0;
            c[e].load(a.cos + pos * a.Dh + d, half);
            sn[e].load(a.sin + pos * a.Dh + d, half);
        }
        if (i >= a.H * a.per) return;
#pragma unroll
        for (int e = 0; e < kRows; e++) {
            if (!of[e].ok) continue;
            Item<HV> it;
            it.rotated(x[e], c[e], sn[e]);
            half_t *to = a.q_out + (int64_t)(row0 + e) * a.ldqo + h * a.Dh + d;
            // an item that reaches back writes its own columns only: the others may be the input's, which another thread has yet to read
            const int own = (i - i / a.per * a.per) * HV - d;
            if (own == 0) {
                put<HV>(to, it.a, 1.f);
                put<HV>(to + half, it.b, 1.f);
            } else
#pragma unroll
                for (int k = 2; k < HV; k += 2)            // (own and the columns are even)
                    if (k >= own) {
                        *reinterpret_cast<half2_t *>(to + k) = half2_t{f2h(it.a[k]), f2h(it.a[k + 1])};
                        *reinterpret_cast<half2_t *>(to + half + k) = half2_t{f2h(it.b[k]), f2h(it.b[k + 1])};
                    }
        }
        return;
    }
    if ((int)blockIdx.x >= pages) {
        const int b = ((int)blockIdx.x - pages) * 64 + (int)threadIdx.x;
        if (threadIdx.x < 64 && b < pb.B && !sequence(pb, b, limit, a.max_new).ok) report(pb, b);
        return;
    }
    // heads of a page next to each other on an XCD: they share 128-byte lines of the rows
    const int chunk = pages / 8, number = (int)blockIdx.x < 8 * chunk ? (int)(blockIdx.x & 7) * chunk + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
    const int x = number / a.Hkv, h = number - x * a.Hkv;
    int unit;
    const int b = a.units.find(pb, x, &unit);
    if (b >= pb.B) return;
    const Sequence s = sequence(pb, b, limit, a.max_new);
    if (!s.ok || s.n <= 0) return;
    const int pi = s.first / pb.page + unit, p0 = max(s.first, pi * pb.page), m = min(s.first + s.n, (pi + 1) * pb.page) - p0;
    if (m <= 0) return;
    const int id = pb.table[(int64_t)b * pb.ldt + pi];
    // the rows, requested with the page's number
    const int t0 = s.s0 + p0 - s.first, items = m * a.per;
    const half_t *kr = a.k + (int64_t)t0 * a.ldk + h * a.Dh, *vr = a.v + (int64_t)t0 * a.ldv + h * a.Dh;
    Loaded<HV> k[2], v[2], c[2], sn[2];
    int at[2];                                 // where the item goes, elements from the first row's slot
    const int Dp = padded_dim(a.Dh);
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int i = min((int)threadIdx.x + e * T, items - 1), t = (int)((unsigned)i * a.per_magic >> 16), d = column(i - t * a.per);
        at[e] = t * Dp + d;
        k[e].load(kr + t * a.ldk + d, half);
        c[e].load(a.cos + (int64_t)(p0 + t) * a.Dh + d, half);
        sn[e].load(a.sin + (int64_t)(p0 + t) * a.Dh + d, half);
        v[e].load(vr + t * a.ldv + d, half);
    }
    if (id < 0 || id >= pb.P) {
        if (threadIdx.x == 0) report(pb, b);
        return;
    }
    const int slot0 = p0 - pi * pb.page;
    const int64_t ph = (int64_t)id * a.Hkv + h;
    P *kp = (P *)a.k_pages + ph * pb.page * Dp, *vp = (P *)a.v_pages + ph * pb.page * Dp;
    float was_k = 0.f, was_v = 0.f, inv_k = 1.f, inv_v = 1.f;
    if (sizeof(P) == 1 && slot0 > 0) {
        was_k = a.k_scale[ph];
        was_v = a.v_scale[ph];
    }
    Item<HV> ik[2], iv[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        ik[e].rotated(k[e], c[e], sn[e]);
        iv[e].plain(v[e]);
    }
    if constexpr (sizeof(P) == 1) {
        float mk = fmaxf(ik[0].amax(), ik[1].amax()), mv = fmaxf(iv[0].amax(), iv[1].amax());      // (a last one twice is no matter)
        mk = wave_max(mk);
        mv = wave_max(mv);
        if constexpr (T > 64) {
            __shared__ float red[T / 64][2];
            if ((threadIdx.x & 63) == 0) {
                red[threadIdx.x >> 6][0] = mk;
                red[threadIdx.x >> 6][1] = mv;
            }
            __syncthreads();                   // (everyone has read the old scales, too)
#pragma unroll
            for (int w = 0; w < T / 64; w++) {
                mk = fmaxf(mk, red[w][0]);
                mv = fmaxf(mv, red[w][1]);
            }
        }
        const float to_k = rescale<T>((uint8_t *)kp, slot0, Dp, mk, was_k), to_v = rescale<T>((uint8_t *)vp, slot0, Dp, mv, was_v);
        if (threadIdx.x == 0) {
            a.k_scale[ph] = to_k;
            a.v_scale[ph] = to_v;
        }
        inv_k = 1.f / to_k;
        inv_v = 1.f / to_v;
    }
    kp += slot0 * Dp;
    vp += slot0 * Dp;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        if ((int)threadIdx.x + e * T >= items) break;
        put<HV>(kp + at[e], ik[e].a, inv_k);
        put<HV>(kp + at[e] + half, ik[e].b, inv_k);
        put<HV>(vp + at[e], iv[e].a, inv_v);
        put<HV>(vp + at[e] + half, iv[e].b, inv_v);
    }
    // the padding of the rows, four columns at a time
    const int pad = (Dp - a.Dh) / 4;
    for (int i = threadIdx.x; i < m * pad; i += T) {
        const int t = i / pad, d = t * Dp + a.Dh + (i - t * pad) * 4;
        typedef P four_t __attribute__((ext_vector_type(4)));
        *reinterpret_cast<four_t *>(kp + d) = four_t{};
        *reinterpret_cast<four_t *>(vp + d) = four_t{};
    }
}

template <int T, int HV, class P>
int launch(AppendArgs a, hipStream_t st)
{
    constexpr int TQ = T < 256 ? T : 256, kRows = rows_of<T>();
    a.slices = (a.H * a.per + TQ - 1) / TQ;
    const int64_t rows = a.q ? ((int64_t)a.pb.T + kRows - 1) / kRows * a.slices : 0;
    const int64_t grid = a.units.count * a.Hkv + (a.pb.B + 63) / 64 + (rows + T / TQ - 1) / (T / TQ);
    CACTI_REQUIRE(grid * T <= UINT32_MAX, CACTI_E_NOTIMPL, "paged_append: too many pages or rows in one call");
    hipLaunchKernelGGL((paged_append_kernel<T, HV, P>), dim3((unsigned)grid), dim3(T), 0, st, a);
    return launch_status("paged_append");
}
// As many threads as hold the rows of a page in one call, two items each
template <int HV, class P>
int launch(const AppendArgs &a, hipStream_t st)
{
    const int items = (a.max_new < a.pb.page ? a.max_new : a.pb.page) * a.per;
    return items <= 128 ? launch<64, HV, P>(a, st) : items <= 512 ? launch<256, HV, P>(a, st) : launch<1024, HV, P>(a, st);
}

}  // namespace

CACTI_API int cacti_hip_paged_append(int64_t T, int64_t B, int64_t H, int64_t Hkv, int64_t Dh, int64_t max_new, const void *q, int64_t ldq,
                                     const void *k, int64_t ldk, const void *v, int64_t ldv, const void *cos16, const void *sin16,
                                     int64_t n_pos, void *q_rot, int64_t ldqr, void *k_pages, void *v_pages, void *k_scale, void *v_scale,
                                     int bits, int64_t P, int64_t page, const void *table, int64_t ldt, int64_t W, const void *starts,
                                     const void *lens, void *status, void *stream)
{
    PagedBatch pb;
    const int rc = paged_batch("paged_append", T, B, H, Hkv, Dh, max_new, table, ldt, W, starts, lens, status, k_pages, v_pages, k_scale,
                               v_scale, bits, P, page, &pb);
    if (rc) return rc;
    CACTI_REQUIRE(k && v && cos16 && sin16 && n_pos > 0 && !q == !q_rot, CACTI_E_INVALID, "paged_append: null pointer");
    CACTI_REQUIRE(ldk >= Hkv * Dh && ldv >= Hkv * Dh && (!q || (ldq >= H * Dh && ldqr >= H * Dh)), CACTI_E_INVALID,
                  "paged_append: row pitch below a row");
    CACTI_REQUIRE(ldk % 4 == 0 && ldv % 4 == 0 && (!q || (ldq % 4 == 0 && ldqr % 4 == 0)) && aligned(k, 8) && aligned(v, 8) && aligned(q, 8) &&
                      aligned(q_rot, 8) && aligned(cos16, 8) && aligned(sin16, 8),
                  CACTI_E_INVALID, "paged_append: operands must be 8-byte aligned with row pitches that are multiples of 4");
    // queries in place: a workgroup reads what it writes; anything else that is written here another may yet have to read
    CACTI_REQUIRE(!q || ((q == q_rot && (ldq == ldqr || T == 1)) || !rows_share(T, q, ldq, H * Dh, q_rot, ldqr, H * Dh)), CACTI_E_INVALID,
                  "paged_append: the rotated queries take the queries' place, with the same pitch, or share no memory with them");
    CACTI_REQUIRE(!q || (!rows_share(T, k, ldk, Hkv * Dh, q_rot, ldqr, H * Dh) && !rows_share(T, v, ldv, Hkv * Dh, q_rot, ldqr, H * Dh)),
                  CACTI_E_INVALID, "paged_append: the rotated queries share memory with the keys or values");
    if (max_new > T) max_new = T;
    // n rows touch up to (n + page - 2) / page + 1 pages, which is no more than n / page + 2
    const Units units = make_units(T, B, page, 1, 2, (max_new + page - 2) / page + 1);
    const int HV = Dh >= 16 ? 8 : 2, per = (int)((Dh / 2 + HV - 1) / HV);
    const AppendArgs a = {pb,   units, (int)H,           (int)Hkv, (int)Dh, (int)max_new, per, 0, 65536u / per + 1, n_pos, (const half_t *)q,
                          (const half_t *)k, (const half_t *)v, (const half_t *)cos16, (const half_t *)sin16, ldq, ldk, ldv, ldqr,
                          (half_t *)q_rot, k_pages, v_pages, (float *)k_scale, (float *)v_scale};
    hipStream_t st = (hipStream_t)stream;
    if (HV == 8) return bits == 8 ? launch<8, uint8_t>(a, st) : launch<8, half_t>(a, st);
    return bits == 8 ? launch<2, uint8_t>(a, st) : launch<2, half_t>(a, st);
}
