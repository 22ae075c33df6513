// Verification of drafted tokens (speculative decoding): which of the tokens that a drafting model proposed the target model's
// probabilities keep, and the token that follows them, from random numbers that the caller gives.
//
// Rows s .. s + n - 1 of a sequence are its last token and the n - 1 drafted ones; row i's logits say what follows it, so the
// drafted token x_i is the token of row i + 1.  With p = softmax(target / T), q = softmax(draft / T) (one-hot at x_i where the
// drafting model has no probabilities or T = 0; p is one-hot at the first arg max then):
//   x_i is kept if u_i q_i(x_i) < p_i(x_i);  a = the first that is not, or n - 1
//   w = max(p_a - q_a, 0) if a < n - 1, p_a else;  next token = the least j with sum_{i <= j} w_i > r sum w
// The tokens that are kept followed by that one are distributed as the target model's own.
//
// Exponentials and sums are fp64: what is drawn goes by on which side of a border of the running sum r lies, and with sums that
// are off by e of their total some V e of all draws come out differently (32000 tokens, fp32 sums: one in several hundred).
// That arithmetic, some 17 operations of 64 bits a logit, bounds the first launch (twice the time that its bytes take), which is half of a
// batch; the other half is the latency of the two launches behind it.
//
// Three launches, each as wide as its work.  A row is cut into entries of 2048 logits, one to a wave, which needs no barrier and
// spreads five rows over 20 workgroups: their maxima and sums relative to them, of every row of both models.  Then workgroups of
// each sequence form the rows' sums from them, see which drafted tokens are kept and sum what is left of p in the first row whose
// token is not, 512 logits to a wave.  Then a workgroup of each sequence finds the entry in which r lies and the token in it.
// us, five rows of 32000 with a drafting model / 64 sequences, 310 rows: 16.7 / 33.3, of which the first launch is 4 / 18; the same batch
// without the drafting model's logits 23.4, greedy (two launches) 9.9.  A
// workgroup per row that drew for every row that might end its sequence 77 / 115, one per sequence for the last two steps 22.5 / 38.6;
// the last step by the last of a sequence's workgroups to write, which takes fences between the XCDs, 18.1 / 116.
#include "operands.h"
#include "vocab_row.h"

using namespace cacti;

namespace {

constexpr int kRounds = 4, kPieces = 64 * kRounds;         // 16-byte pieces of an entry
constexpr int kLeft = 64;                      // of an entry of what is left of p
constexpr int kEntryWaves = 4;                 // entries of a workgroup of the first kernel
constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kDraw = 1024;                    // lanes of the last kernel: two logits each

struct __attribute__((aligned(16))) Entry {
    double z;                                  // sum of exponentials relative to the entry's maximum; greedy: its first arg max
    double m;
};
// The row that ends a sequence, -1 where its numbers do not fit together
struct Head {
    int row, residual, x;                           // whether a drafted token was not kept, which
    float mt, md;
    double it, id;                             // 1 / sums
};

struct VerifyArgs {
    int T, B, V, E, E2;                        // E, E2: entries of a row, of what is left of p
    const half_t *target, *draft;
    int64_t ldt, ldd;
    const uint16_t *tok;
    const int *starts;
    const float *u, *r;
    double c;                                  // log2 e / temperature
    Entry *entries;                            // [2][T][E]: target, draft
    double *left;                              // [B][E2]: sums of what is left of p
    Head *heads;
    int *accepted;
    uint16_t *next;
    int *status;
};

// 2^t for -2^31 < t <= 0: t = n + f, |f| <= 1/2, a polynomial of degree 9 in f (Chebyshev interpolation on that interval,
// 2e-14) and n added to its exponent
__device__ __forceinline__ double exp2_neg(double t)
{
    const double magic = 0x1.8p52, s = t + magic, f = t - (s - magic);        // the sum's low word is n
    double p = 1.0205905724567723e-07;
    p = __builtin_fma(p, f, 1.3259645239858464e-06);
    p = __builtin_fma(p, f, 1.5252672923029364e-05);
    p = __builtin_fma(p, f, 0.00015403433751274572);
    p = __builtin_fma(p, f, 0.0013333558200798331);
    p = __builtin_fma(p, f, 0.0096181291939342831);
    p = __builtin_fma(p, f, 0.055504108664651643);
    p = __builtin_fma(p, f, 0.24022650695640341);
    p = __builtin_fma(p, f, 0.69314718055994617);
    p = __builtin_fma(p, f, 1.0000000000000135);
    return __builtin_amdgcn_ldexp(p, (int)__builtin_bit_cast(uint64_t, s));
}
constexpr double kNothing = 1e-290;            // weights below that are nothing

// A NaN is never chosen
__device__ __forceinline__ float clean(half_t x) { return fmaxf(h2f(x), -INFINITY); }
// 2^((x - mx) c), 0 of -inf; of a maximum that is an infinity 1 for those that are it, 0 for the others
__device__ __forceinline__ double weight(float x, float mx, double c)
{
    const bool fine = fabsf(mx) < INFINITY;
    const float y = fine ? x : x == mx ? 0.f : -INFINITY;
    const double w = exp2_neg(__builtin_fma(y > -INFINITY ? (double)y : 0., c, fine ? -(double)mx * c : 0.));
    return y > -INFINITY ? w : 0.;
}

template <bool GREEDY>
__global__ void __launch_bounds__(64 * kEntryWaves) verify_entries_kernel(VerifyArgs a)
{
    const int row = blockIdx.x, e = blockIdx.y * kEntryWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool drafting = blockIdx.z == 1;
    if (e >= a.E) return;
    const VocabRow t(drafting ? a.draft + row * a.ldd : a.target + row * a.ldt, a.V);
    Entry *to = a.entries + ((int64_t)blockIdx.z * a.T + row) * a.E + e;
    h8 v[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; r++) {
        const int c = e * kPieces + r * 64 + lane;
        if (c < t.pieces()) v[r] = t.load(c, (half_t)-INFINITY);
        else
#pragma unroll
            for (int k = 0; k < 8; k++) v[r].v[k] = (half_t)-INFINITY;
    }
    if (drafting) {                            // a sequence's last row has no drafted token behind it
        bool last = false;
        for (int i = 1 + lane; i <= a.B; i += 64) last = last || a.starts[i] == row + 1;
        if (__ballot(last)) return;
    }
    half2_t h[kRounds * 4], m2 = {(half_t)-INFINITY, (half_t)-INFINITY};      // two at a time; a NaN is no maximum
    __builtin_memcpy(h, v, sizeof(v));
#pragma unroll
    for (int i = 0; i < kRounds * 4; i++) m2 = __builtin_elementwise_max(m2, h[i]);
    const float mx = wave_max(fmaxf(h2f(m2[0]), h2f(m2[1])));
    double z = 0.;
    if (GREEDY) {
        int at = 65536;
#pragma unroll
        for (int r = kRounds - 1; r >= 0; r--)
#pragma unroll
            for (int k = 7; k >= 0; k--) {
                const int j = t.first(e * kPieces + r * 64 + lane) + k;
                if (j >= 0 && j < a.V && clean(v[r].v[k]) == mx) at = j;
            }
        z = -(double)wave_max(-(float)at);
    } else {
        const half_t lowest = (half_t)-65504.f;
        if (fabsf(mx) < INFINITY && (-65504. - (double)mx) * a.c < -1000.) {
            // -inf and a NaN count as the lowest number, which has no weight here
            const double b = -(double)mx * a.c;
#pragma unroll
            for (int i = 0; i < kRounds * 4; i++) {
                const half2_t x = __builtin_elementwise_max(h[i], half2_t{lowest, lowest});
                z += exp2_neg(__builtin_fma((double)h2f(x[0]), a.c, b));
                z += exp2_neg(__builtin_fma((double)h2f(x[1]), a.c, b));
            }
        } else {
#pragma unroll 1
            for (int r = 0; r < kRounds; r++) {
                const int c = e * kPieces + r * 64 + lane;
#pragma unroll 1
                for (int j = t.first(c); c < t.pieces() && j < t.first(c) + 8; j++)
                    if (j >= 0 && j < a.V) z += weight(clean(t.row[j]), mx, a.c);
            }
        }
        z = wave_sum_f64(z);
    }
    if (lane == 0) *to = Entry{z, (double)mx};
}

// A row's maximum and sum, by a wave (with no more than 64 entries)
struct RowSum {
    float m;
    double z;
};
__device__ __forceinline__ RowSum row_sum(const VerifyArgs &a, const Entry *en)
{
    const int lane = threadIdx.x & 63;
    const Entry none = {0., -INFINITY}, e = lane < a.E ? en[lane] : none;
    RowSum s;
    s.m = wave_max((float)e.m);
    s.z = wave_sum_f64(e.z * weight((float)e.m, s.m, a.c));
    return s;
}

// The rows of sequence b up to the first that ends it, a wave to each; `ends` says whether a row does.  Returns that row.
template <class F>
__device__ __forceinline__ int first_end(int s0, int s1, int *stops, F ends)
{
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i0 = s0;; i0 += kWaves) {
        const int row = i0 + wid;
        const bool stop = row >= s1 || ends(row, wid);
        __syncthreads();
        if (lane == 0) stops[wid] = stop;
        __syncthreads();
        for (int w = 0; w < kWaves; w++)
            if (stops[w]) return i0 + w;       // (s1 - 1 ends, so this is below s1)
    }
}

__device__ __forceinline__ bool rows_of(const VerifyArgs &a, int b, int *s0, int *s1)
{
    *s0 = a.starts[b];
    *s1 = a.starts[b + 1];
    return *s0 >= 0 && *s1 <= a.T && *s1 > *s0;
}

// What follows: next[s0 .. s1 - 1] and accepted[b], of row `end` that ends the sequence and the token behind it; by NT lanes
template <int NT>
__device__ __forceinline__ void write_out(const VerifyArgs &a, int b, int s0, int s1, int end, int token)
{
    for (int i = s0 + threadIdx.x; i < s1; i += NT) a.next[i] = i < end ? a.tok[i + 1] : i == end ? (uint16_t)token : (uint16_t)0;
    if (threadIdx.x == 0) a.accepted[b] = end - s0;
}

// The code of the next kernel runs once per lane or a few times, so it is short: what is unrolled is fetched from memory for
// one use (16 logits of both models unrolled, in three places, were 49 KB and some 20 us).

// What is left of p = softmax(target) where the drafting model's q has been taken off, or the token that was drafted
struct Left {
    const half_t *t, *d;                       // d null: none
    float mt, md;
    double it, id, c;
    int x, V;
    __device__ __forceinline__ Left(const VerifyArgs &a, const Head &h)
        : t(a.target + h.row * a.ldt), d(a.draft && h.residual ? a.draft + h.row * a.ldd : nullptr), mt(h.mt), md(h.md), it(h.it), id(h.id),
          c(a.c), x(h.x), V(a.V)
    {
    }
    // of logit j, whose logits are ht and hd
    __device__ __forceinline__ double operator()(half_t ht, half_t hd, int j, bool residual) const
    {
        double y = weight(clean(ht), mt, c) * it;
        if (residual) {
            if (d) y -= weight(clean(hd), md, c) * id;
            else if (j == x) y = 0.;
        }
        return j >= 0 && j < V && y > kNothing ? y : 0.;
    }
};

// Eight halves, the first taken off at a time
struct Eight {
    uint64_t lo, hi;
    __device__ __forceinline__ explicit Eight(const h8 &v)
    {
        uint64_t w[2];
        __builtin_memcpy(w, &v, 16);
        lo = w[0];
        hi = w[1];
    }
    __device__ __forceinline__ half_t take()
    {
        const half_t x = __builtin_bit_cast(half_t, (uint16_t)lo);
        lo = lo >> 16 | hi << 48;
        hi >>= 16;
        return x;
    }
};

// The first of a block's lanes that `hit`s, else (by a rounding) the last that has any weight: lane numbers, by LDS
__device__ __forceinline__ int pick_lane(bool hit, bool any, int *first, int *last)
{
    if (threadIdx.x == 0) *first = INT32_MAX, *last = 0;
    __syncthreads();
    const uint64_t h = __ballot(hit), y = __ballot(any);
    if ((threadIdx.x & 63) == 0) {
        if (h) atomicMin(first, (int)threadIdx.x + __ffsll((unsigned long long)h) - 1);
        if (y) atomicMax(last, (int)threadIdx.x + 63 - __clzll((long long)y));
    }
    __syncthreads();
    return *first < INT32_MAX ? *first : *last;
}

__global__ void __launch_bounds__(kThreads) verify_rows_kernel(VerifyArgs a)
{
    __shared__ int stops[kWaves];
    __shared__ Head found[kWaves];
    const int b = blockIdx.y, wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int s0, s1;
    if (!rows_of(a, b, &s0, &s1)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.heads[b].row = -1;
            if (s1 != s0 && a.status) atomicMax(a.status, 1);
        }
        return;
    }
    const int row = first_end(s0, s1, stops, [&](int i, int w) {
        const bool last = i + 1 >= s1, drafted = a.draft && !last;
        const int x = last ? 0 : a.tok[i + 1], at = min(x, a.V - 1);
        const bool bad = x >= a.V;
        // (the drafted token's logits requested with the sums, not behind them)
        const float xt = clean(a.target[i * a.ldt + at]), xd = drafted ? clean(a.draft[i * a.ldd + at]) : 0.f, u = a.u[i];
        const RowSum t = row_sum(a, a.entries + (int64_t)i * a.E);
        RowSum d = {0.f, 1.};
        if (drafted) d = row_sum(a, a.entries + ((int64_t)a.T + i) * a.E);
        const double it = 1. / t.z, id = 1. / d.z;
        if (lane == 0) found[w] = Head{i, !last, x, t.m, d.m, it, id};
        if (bad && lane == 0 && a.status) atomicMax(a.status, i + 2);
        const double q = drafted ? weight(xd, d.m, a.c) * id : 1.;
        return last || bad || !((double)u * q < weight(xt, t.m, a.c) * it);
    });
    const Head h = found[(row - s0) & (kWaves - 1)];
    if (blockIdx.x == 0 && threadIdx.x == 0) a.heads[b] = h;
    const int e = blockIdx.x * kWaves + wid;
    if (!h.residual || e >= a.E2) return;      // (the entries' sums of p are there)
    const Left lf(a, h);
    const VocabRow t(lf.t, a.V);
    const bool alike = lf.d && ((reinterpret_cast<uintptr_t>(lf.d) ^ reinterpret_cast<uintptr_t>(lf.t)) & 15) == 0;
    const int p = e * kLeft + lane, j0 = t.first(p);
    h8 v = {}, u = {};
    if (p < t.pieces()) {
        v = t.load(p, (half_t)0.f);
        if (alike && t.whole(p)) u = ld8(lf.d + j0);
        else if (lf.d)
#pragma unroll
            for (int k = 0; k < 8; k++) u.v[k] = lf.d[min(max(j0 + k, 0), a.V - 1)];
    }
    Eight v8(v), u8(u);
    double sum = 0.;
#pragma unroll 2
    for (int k = 0; k < 8; k++) sum += lf(v8.take(), u8.take(), j0 + k, true);
    sum = wave_sum_f64(sum);
    if (lane == 0) a.left[(int64_t)b * a.E2 + e] = sum;
}

__global__ void __launch_bounds__(kDraw) verify_draw_kernel(VerifyArgs a)
{
    __shared__ double waves[kDraw / 64];
    __shared__ int first, last, token;
    const int b = blockIdx.x, wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Head h = a.heads[b];
    const int s0 = a.starts[b], s1 = a.starts[b + 1];
    const double r = (double)a.r[b];
    if (h.row < 0) {
        if (threadIdx.x == 0) a.accepted[b] = 0;
        return;
    }
    auto block_scan = [&](double v, double *total) {
        const double in = scan_f64(v);
        __syncthreads();
        if (lane == 63) waves[wid] = in;
        __syncthreads();
        double before = 0.;
        *total = 0.;
        for (int w = 0; w < kDraw / 64; w++) {
            if (w == wid) before = *total;
            *total += waves[w];
        }
        return in + before;
    };
    // the entry in which r lies, one to a lane
    const int en = threadIdx.x;
    double mine = en < a.E2 && h.residual ? a.left[(int64_t)b * a.E2 + en] : 0., total;
    double upto = block_scan(mine, &total);
    const bool residual = h.residual && total > kNothing;        // p = q: nothing is left of it
    if (!residual) {
        mine = 0.;
        if (en < a.E) {
            const Entry x = a.entries[(int64_t)h.row * a.E + en];
            mine = x.z * weight((float)x.m, h.mt, a.c) * h.it;
        }
        upto = block_scan(mine, &total);
    }
    const double want = r * total;
    const int e = pick_lane(mine > kNothing && upto > want, mine > kNothing, &first, &last);
    if ((int)threadIdx.x == e) waves[0] = upto - mine;
    __syncthreads();
    const double before = waves[0];
    // the token in it, two to a lane
    const Left lf(a, h);
    const VocabRow t(lf.t, a.V);
    const int size = 8 * (residual ? kLeft : kPieces), j0 = t.first(e * size / 8), j = j0 + 2 * (int)threadIdx.x;
    double w[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int at = min(max(j + k, 0), a.V - 1);
        w[k] = lf(t.row[at], lf.d ? lf.d[at] : (half_t)0.f, 2 * (int)threadIdx.x < size ? j + k : -1, residual);
    }
    mine = w[0] + w[1];
    upto = block_scan(mine, &total) + before;
    const int lane_of = pick_lane(mine > 0. && upto > want, mine > 0., &first, &last);
    if ((int)threadIdx.x == lane_of) token = j + !(w[0] > 0. && (upto - w[1] > want || !(w[1] > 0.)));
    __syncthreads();
    write_out<kDraw>(a, b, s0, s1, h.row, min(max(token, 0), a.V - 1));
}

__global__ void __launch_bounds__(kThreads) verify_greedy_kernel(VerifyArgs a)
{
    __shared__ int stops[kWaves];
    __shared__ int found[kWaves];
    const int b = blockIdx.x, lane = threadIdx.x & 63;
    int s0, s1;
    if (!rows_of(a, b, &s0, &s1)) {
        if (threadIdx.x == 0) {
            a.accepted[b] = 0;
            if (s1 != s0 && a.status) atomicMax(a.status, 1);
        }
        return;
    }
    const int row = first_end(s0, s1, stops, [&](int i, int w) {
        const bool last = i + 1 >= s1;
        const int x = last ? 0 : a.tok[i + 1];
        const float u = a.u[i];
        const Entry none = {65536., -INFINITY}, e = lane < a.E ? a.entries[(int64_t)i * a.E + lane] : none;
        const double m = wave_max((float)e.m);
        const int at = (int)-wave_max(e.m == m ? -(float)e.z : -65536.f);
        if (lane == 0) found[w] = at;
        if (x >= a.V && lane == 0 && a.status) atomicMax(a.status, i + 2);
        return last || x != at || !(u < 1.f);
    });
    write_out<kThreads>(a, b, s0, s1, row, found[(row - s0) & (kWaves - 1)]);
}

int64_t entries_of(int64_t V, int size) { return ((V + 14) / 8 + size - 1) / size; }        // wherever a row begins

}  // namespace

CACTI_API size_t cacti_hip_verify_draft_workspace(int64_t T, int64_t B, int64_t V)
{
    if (T <= 0 || B <= 0 || V <= 0) return 0;
    return (size_t)(2 * T * entries_of(V, kPieces)) * sizeof(Entry) + (size_t)B * (sizeof(Head) + (size_t)entries_of(V, kLeft) * 8);
}

CACTI_API int cacti_hip_verify_draft_f16(int64_t T, int64_t B, int64_t V, const void *target, int64_t ldt, const void *draft, int64_t ldd,
                                         const void *tok, const void *starts, const void *u, const void *r, double temperature, void *accepted,
                                         void *next, void *workspace, size_t workspace_bytes, void *status, void *stream)
{
    CACTI_REQUIRE(T > 0 && B > 0 && V > 0, CACTI_E_INVALID, "verify_draft: empty shape");
    CACTI_REQUIRE(target && tok && starts && u && r && accepted && next && workspace, CACTI_E_INVALID, "verify_draft: null pointer");
    CACTI_REQUIRE(V <= 65536 && T < (1 << 18) && B <= 65535, CACTI_E_NOTIMPL, "verify_draft: at most 65536 tokens, 2^18 rows, 65535 sequences");
    CACTI_REQUIRE(ldt >= V && (!draft || ldd >= V), CACTI_E_INVALID, "verify_draft: row pitch below a row");
    CACTI_REQUIRE(temperature >= 0. && temperature <= 1e6 && (temperature == 0. || temperature >= 1e-3), CACTI_E_INVALID,
                  "verify_draft: the temperature is 0 or from 1e-3 to 1e6");
    CACTI_REQUIRE(aligned(target, 2) && aligned(draft, 2) && aligned(tok, 2) && aligned(next, 2) && aligned(starts, 4) && aligned(u, 4) &&
                      aligned(r, 4) && aligned(accepted, 4) && aligned(workspace, 16) && aligned(status, 4),
                  CACTI_E_INVALID, "verify_draft: misaligned operand");
    CACTI_REQUIRE(workspace_bytes >= cacti_hip_verify_draft_workspace(T, B, V), CACTI_E_INVALID, "verify_draft: workspace too small");
    CACTI_REQUIRE(!rows_share(1, tok, T, T, next, T, T), CACTI_E_INVALID, "verify_draft: the tokens behind the rows share memory with theirs");
    const bool greedy = temperature == 0.;
    const int64_t E = entries_of(V, kPieces), E2 = entries_of(V, kLeft);
    Entry *entries = (Entry *)workspace;
    Head *heads = (Head *)(entries + 2 * T * E);
    const VerifyArgs a = {(int)T, (int)B, (int)V, (int)E, (int)E2, (const half_t *)target, greedy ? nullptr : (const half_t *)draft, ldt, ldd,
                          (const uint16_t *)tok, (const int *)starts, (const float *)u, (const float *)r,
                          greedy ? 0. : 1.4426950408889634 / temperature, entries, (double *)(heads + B), heads, (int *)accepted,
                          (uint16_t *)next, (int *)status};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)T, (unsigned)((E + kEntryWaves - 1) / kEntryWaves), a.draft ? 2 : 1), block(64 * kEntryWaves);
    if (greedy) hipLaunchKernelGGL(verify_entries_kernel<true>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(verify_entries_kernel<false>, grid, block, 0, st, a);
    int rc = launch_status("verify_draft");
    if (rc) return rc;
    if (greedy) {
        hipLaunchKernelGGL(verify_greedy_kernel, dim3((unsigned)B), dim3(kThreads), 0, st, a);
        return launch_status("verify_draft (greedy)");
    }
    hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)((E2 + kWaves - 1) / kWaves), (unsigned)B), dim3(kThreads), 0, st, a);
    rc = launch_status("verify_draft (rows)");
    if (rc) return rc;
    hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)B), dim3(kDraw), 0, st, a);
    return launch_status("verify_draft (draw)");
}
