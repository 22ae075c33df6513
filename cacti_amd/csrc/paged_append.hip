// New keys and values into the pages of a cache, rotated on the way, with the queries of the same rows.
//
//   k'[d] = k[d] cos[p][d] - k[d + Dh/2] sin[p][d]   (d < Dh/2; the other half: k[d] cos[p][d] + k[d - Dh/2] sin[p][d])
// with the products exact (22 of 24 bits) and one rounding of their sum in fp32, then one into the page: to f16, or to e4m3
// of k' / scale with the scale 2^e of the page and head.  A power of two costs the quotient no rounding and e4m3 nothing of
// its precision (it has an exponent of its own), and codes that are there already can be carried over to a larger scale
// exactly, but for those that become subnormal.
//
// A workgroup owns a page and a head: it looks at the new rows of that page, takes the least scale that holds them and no
// less than that of older rows, codes those again where it grew, and writes.  No other workgroup touches that page and head.
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
    CACTI_REQUIRE(T <= INT32_MAX / H && B < 65536 * 16 && P <= INT32_MAX && W <= INT32_MAX / page && H <= 4096 && ldt >= W, CACTI_E_NOTIMPL,
                  "%s: too many rows, sequences or pages, or a table pitch below its width", who);
    CACTI_REQUIRE(aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(table, 4) && aligned(starts, 4) && aligned(lens, 4) &&
                      aligned(k_scale, 4) && aligned(v_scale, 4) && aligned(status, 4),
                  CACTI_E_INVALID, "%s: pages must be 16-byte aligned", who);
    *pb = {(int)T, (int)B, (int)page, (int)W, ldt, (int)P, (const int *)starts, (const int *)lens, (const int *)table, (int *)status};
    return 0;
}

}  // namespace cacti

namespace {

constexpr int kThreads = 256;
constexpr int kMinExp = -32, kMaxExp = 15;     // of a page's scale: 2^-24 / 448 and beyond sqrt(2) 65504 / 448

struct AppendArgs {
    PagedBatch pb;
    Units units;
    int H, Hkv, Dh, max_new;
    int64_t n_pos;                             // rows of cos, sin
    const half_t *q, *k, *v, *cos, *sin;
    int64_t ldq, ldk, ldv, ldqo;
    half_t *q_out;
    void *k_pages, *v_pages;
    float *k_scale, *v_scale;
};

template <int HV>
struct __attribute__((aligned(2 * HV))) hv {
    half_t v[HV];
};

// HV columns of the left half of a head from d on and their partners in the right half, rotated (or, ROT false, as they are)
template <int HV, bool ROT>
struct Item {
    float a[HV], b[HV];
    __device__ __forceinline__ Item(const half_t *x, const half_t *c, const half_t *s, int half)
    {
        const hv<HV> x0 = *reinterpret_cast<const hv<HV> *>(x), x1 = *reinterpret_cast<const hv<HV> *>(x + half);
        if (ROT) {
            const hv<HV> c0 = *reinterpret_cast<const hv<HV> *>(c), c1 = *reinterpret_cast<const hv<HV> *>(c + half);
            const hv<HV> s0 = *reinterpret_cast<const hv<HV> *>(s), s1 = *reinterpret_cast<const hv<HV> *>(s + half);
#pragma unroll
            for (int i = 0; i < HV; i++) {
                a[i] = h2f(x0.v[i]) * h2f(c0.v[i]) - h2f(x1.v[i]) * h2f(s0.v[i]);
                b[i] = h2f(x1.v[i]) * h2f(c1.v[i]) + h2f(x0.v[i]) * h2f(s1.v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < HV; i++) {
                a[i] = h2f(x0.v[i]);
                b[i] = h2f(x1.v[i]);
            }
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
    hv<HV> h;
#pragma unroll
    for (int i = 0; i < HV; i++) h.v[i] = f2h(x[i]);
    *reinterpret_cast<hv<HV> *>(to) = h;
}
// e4m3, to nearest, ties to even; NaN and infinities become NaN
template <int HV>
__device__ __forceinline__ void put(uint8_t *to, const float (&x)[HV], float inv)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inv, x[1] * inv, 0, false);
    if (HV == 4) w = __builtin_amdgcn_cvt_pk_fp8_f32(x[HV - 2] * inv, x[HV - 1] * inv, w, true);
    if (HV == 4) *reinterpret_cast<int *>(to) = w;
    else *reinterpret_cast<uint16_t *>(to) = (uint16_t)w;
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

// The rows t0 .. t0 + m - 1 of one of k, v into the slots from slot0 on.  page: the page's rows of this head
template <int HV, bool ROT, class P>
__device__ __forceinline__ void write_rows(const AppendArgs &a, const half_t *x, int64_t ldx, int h, int pos0, int slot0, int m, P *page,
                                           float *scale, float *red)
{
    const int Dh = a.Dh, half = Dh / 2, per = half / HV, Dp = padded_dim(Dh);
    auto item = [&](int i) __attribute__((always_inline)) {
        const int t = i / per, d = (i - t * per) * HV;
        return Item<HV, ROT>(x + (int64_t)t * ldx + h * Dh + d, a.cos + (int64_t)(pos0 + t) * Dh + d, a.sin + (int64_t)(pos0 + t) * Dh + d, half);
    };
    float inv = 1.f;
    if constexpr (sizeof(P) == 1) {
        float mx = 0.f;
        for (int i = threadIdx.x; i < m * per; i += kThreads) mx = fmaxf(mx, item(i).amax());
        mx = block_reduce(mx, OpMax(), 0.f, red);
        float to = scale_for(mx);
        if (slot0 > 0) {
            const float was = *scale;
            if (was >= to) to = was;
            else {
                const float f = was / to;
                for (int i = threadIdx.x; i < slot0 * (Dp / 4); i += kThreads) {
                    int w = reinterpret_cast<int *>(page)[i];
                    const float c0 = __builtin_amdgcn_cvt_f32_fp8(w, 0), c1 = __builtin_amdgcn_cvt_f32_fp8(w, 1);
                    const float c2 = __builtin_amdgcn_cvt_f32_fp8(w, 2), c3 = __builtin_amdgcn_cvt_f32_fp8(w, 3);
                    w = __builtin_amdgcn_cvt_pk_fp8_f32(c0 * f, c1 * f, 0, false);
                    reinterpret_cast<int *>(page)[i] = __builtin_amdgcn_cvt_pk_fp8_f32(c2 * f, c3 * f, w, true);
                }
            }
        }
        __syncthreads();                       // everyone has read the old scale
        if (threadIdx.x == 0) *scale = to;
        inv = 1.f / to;
    }
    for (int i = threadIdx.x; i < m * per; i += kThreads) {
        const Item<HV, ROT> it = item(i);
        const int t = i / per, d = (i - t * per) * HV;
        P *to = page + (slot0 + t) * Dp + d;
        put<HV>(to, it.a, inv);
        put<HV>(to + half, it.b, inv);
    }
    const int pad = (Dp - Dh) / 4;             // the padding of the rows, in pieces of four
    for (int i = threadIdx.x; i < m * pad; i += kThreads) {
        const int t = i / pad, d = Dh + (i - t * pad) * 4;
        P *to = page + (slot0 + t) * Dp + d;
#pragma unroll
        for (int j = 0; j < 4; j++) to[j] = (P)0;
    }
}

// Workgroups: one for each unit (page of a sequence) and head, then one for each row of the queries.
template <int HV, class P>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(AppendArgs a)
{
    __shared__ float red[kThreads / 64];
    const PagedBatch &pb = a.pb;
    const int64_t limit = min((int64_t)pb.W * pb.page, a.n_pos);
    const int64_t pages = a.units.count * a.Hkv;
    if ((int64_t)blockIdx.x >= pages) {
        const int row = (int)(blockIdx.x - pages);
        const int b = count_below(pb.B, row, [&](int i) { return pb.starts[i]; });
        if (b >= pb.B) return;
        const Sequence s = sequence(pb, b, limit, a.max_new);
        if (!s.ok || row < s.s0 || row >= s.s0 + s.n) return;                    // reported by the pages' workgroups
        const int pos = s.first + row - s.s0, half = a.Dh / 2, per = half / HV;
        const half_t *c = a.cos + (int64_t)pos * a.Dh, *sn = a.sin + (int64_t)pos * a.Dh;
        for (int i = threadIdx.x; i < a.H * per; i += kThreads) {
            const int h = i / per, d = (i - h * per) * HV;
            const Item<HV, true> it(a.q + row * a.ldq + h * a.Dh + d, c + d, sn + d, half);
            half_t *to = a.q_out + row * a.ldqo + h * a.Dh + d;
            put<HV>(to, it.a, 1.f);
            put<HV>(to + half, it.b, 1.f);
        }
        return;
    }
    const int64_t x = blockIdx.x / a.Hkv;
    const int h = (int)(blockIdx.x - x * a.Hkv);
    int unit;
    const int b = a.units.find(pb, x, &unit);
    if (b >= pb.B) return;
    const Sequence s = sequence(pb, b, limit, a.max_new);
    if (!s.ok || s.n <= 0) {
        if (!s.ok && threadIdx.x == 0) report(pb, b);
        return;
    }
    const int pi = s.first / pb.page + unit, p0 = max(s.first, pi * pb.page), p1 = min(s.first + s.n, (pi + 1) * pb.page);
    if (p0 >= p1) return;
    const int id = pb.table[(int64_t)b * pb.ldt + pi];
    if (id < 0 || id >= pb.P) {
        if (threadIdx.x == 0) report(pb, b);
        return;
    }
    const int slot0 = p0 - pi * pb.page, t0 = s.s0 + p0 - s.first;
    const int64_t ph = (int64_t)id * a.Hkv + h, at = ph * pb.page * padded_dim(a.Dh);
    write_rows<HV, true>(a, a.k + (int64_t)t0 * a.ldk, a.ldk, h, p0, slot0, p1 - p0, (P *)a.k_pages + at, a.k_scale + ph, red);
    __syncthreads();
    write_rows<HV, false>(a, a.v + (int64_t)t0 * a.ldv, a.ldv, h, p0, slot0, p1 - p0, (P *)a.v_pages + at, a.v_scale + ph, red);
}

template <int HV, class P>
int launch(const AppendArgs &a, int64_t grid, hipStream_t st)
{
    hipLaunchKernelGGL((paged_append_kernel<HV, P>), dim3((unsigned)grid), dim3(kThreads), 0, st, a);
    return launch_status("paged_append");
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
    if (max_new > T) max_new = T;
    // n rows touch up to (n + page - 2) / page + 1 pages, which is no more than n / page + 2
    const Units units = make_units(T, B, page, 2, (max_new + page - 2) / page + 1);
    const int64_t grid = units.count * Hkv + (q ? T : 0);
    CACTI_REQUIRE(grid < (1 << 24), CACTI_E_NOTIMPL, "paged_append: too many pages in one call");
    const AppendArgs a = {pb,   units, (int)H,           (int)Hkv, (int)Dh, (int)max_new, n_pos, (const half_t *)q, (const half_t *)k,
                          (const half_t *)v, (const half_t *)cos16, (const half_t *)sin16, ldq, ldk, ldv, ldqr, (half_t *)q_rot,
                          k_pages, v_pages, (float *)k_scale, (float *)v_scale};
    hipStream_t st = (hipStream_t)stream;
    if (Dh % 8 == 0) return bits == 8 ? launch<4, uint8_t>(a, grid, st) : launch<4, half_t>(a, grid, st);
    return bits == 8 ? launch<2, uint8_t>(a, grid, st) : launch<2, half_t>(a, grid, st);
}
