// Losses over tokens that a model drew itself: their log-probabilities, a clipped policy loss, and a loss over pairs of texts of
// which one is preferred.  With the logits z of a row, its token x and a temperature tau:
//   lp = z_x / tau - log sum_j e^(z_j / tau),   d lp / d z_j = ([j = x] - p_j) / tau
// policy:      r = e^(lp - old),  loss = -min(r A, clip(r, 1 - lo, 1 + hi) A) + beta (e^d - d - 1),  d = ref - lp
//              d loss / d lp = -[r A <= clip(r) A] r A + beta (1 - e^d)
// preference:  s = sum over a text's rows of lp - ref,  h = beta (s_chosen - s_rejected),
//              loss = -(1 - eps) log sigma(h) - eps log sigma(-h)
// A row that a mask leaves out has log-probability, loss and gradient 0, and its logits are not read.
//
// A workgroup to a row, which it holds in registers from one read on.  What a row's gradient of the policy loss is multiplied with
// depends on that row alone, so it is written from the same registers: one read and one write of the logits in all.  The pairs'
// factors depend on whole texts: two reads and one write, and a launch of one workgroup a pair between them.
//
// Bound by memory.  On the device: the policy loss of 2048 rows of 32000, a third of them left out, 40.9 us, 5.4 TB/s of logits read and
// gradient written; pairs of 1666 rows of 32000 15.5 + 5.5 + 26.4 us, 5.0 TB/s; 192 rows of 1024 4.0 us, a launch's own time.  Two
// workgroups and more to a compute unit cover what a row waits for its sums.
#include "operands.h"
#include "vocab_row.h"

using namespace cacti;

namespace {

struct TokenArgs {
    int64_t N;
    int V;
    const half_t *logit;
    int64_t ld, ldd;
    const uint16_t *tok;
    const uint8_t *mask;                       // null, or 0 for a row that is left out
    float inv_temp;
    float *logp, *stats;
    const float *dlogp;
    half_t *grad;
    int acc;
    int *status;
    // of the policy loss
    const float *old, *adv, *ref, *scale;
    float lo, hi, beta;
    float *loss;
};

// The token of a row, or -1 for one that is left out; who: the thread that names a token that there is not
__device__ __forceinline__ int token(const TokenArgs &a, int64_t n, bool who)
{
    if (a.mask && !a.mask[n]) return -1;
    const int x = a.tok[n];
    if (x < a.V) return x;
    if (who && a.status) atomicMax(a.status, (int)n + 1);
    return -1;
}

template <int T>
__device__ __forceinline__ float block_of(float v, bool sum, float *red)
{
    v = sum ? wave_sum(v) : wave_max(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < T / 64; w++) v = sum ? v + red[w] : fmaxf(v, red[w]);
    return v;
}

// Maximum of a row, the sum of its exponentials and the log-probability of a token, the same in all threads and, for rows that
// begin alike behind a 16-byte boundary, in all kernels
struct RowStats {
    float mx, sum, logp;
};
template <int T, int NP>
__device__ __forceinline__ RowStats row_stats(Held<T, NP> &h, float zx, float inv_temp)
{
    __shared__ float red[2][T / 64];
    const float c2 = inv_temp * 1.44269504088896340736f;
    if (h.edge < 0) h.e = (half_t)-INFINITY;
    float mx = fmaxf(zx, h2f(h.e));            // (with the token's: all that is read of the row has come before anybody writes)
    if (h.hi > h.lo) {                         // (what a thread does not have is some other element of the row)
        half8_t m8 = h.x[0];
#pragma unroll
        for (int i = 1; i < NP; i++) m8 = __builtin_elementwise_max(m8, h.x[i]);
#pragma unroll
        for (int k = 0; k < 8; k++) mx = fmaxf(mx, h2f(m8[k]));
    }
    RowStats r;
    r.mx = block_of<T>(mx, false, red[0]);
    float s = __builtin_amdgcn_exp2f((h2f(h.e) - r.mx) * c2);
    s = h.edge < 0 ? 0.f : s;
#pragma unroll
    for (int i = 0; i < NP; i++) {
        if (!h.has(i)) break;                  // (a wave without a piece sums none: 32784 wide 100 us, not 149)
        float p = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) p += __builtin_amdgcn_exp2f((h2f(h.x[i][k]) - r.mx) * c2);
        s += p;
    }
    r.sum = block_of<T>(s, true, red[1]);
    r.logp = (zx - r.mx) * inv_temp - logf(r.sum);
    return r;
}

// gradient = c ([j = x] - e^((z_j - max) / tau) / sum) of the row in h, whose pieces are the gradient's
template <int T, int NP>
__device__ __forceinline__ void put_gradient(const TokenArgs &a, half_t *to, const VocabRow &g, const Held<T, NP> &h, int x, float mx, float sum, float c)
{
    const float c2 = a.inv_temp * 1.44269504088896340736f, q = -c / sum;
    const int px = (x + g.off) / 8, kx = (x + g.off) % 8;
    auto value = [&](half_t z) __attribute__((always_inline)) { return q * __builtin_amdgcn_exp2f((h2f(z) - mx) * c2); };
#pragma unroll
    for (int i = 0; i < NP; i++) {
        if (!h.has(i)) break;
        const int p = h.piece(i);
        float d[8];
#pragma unroll
        for (int k = 0; k < 8; k++) d[k] = value(h.x[i][k]);
        if (p == px)
#pragma unroll
            for (int k = 0; k < 8; k++) d[k] += k == kx ? c : 0.f;
        half8_t o, *at = reinterpret_cast<half8_t *>(to + g.first(p));
        if (a.acc) {
            o = *at;
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = combined(d[k], 1, o[k]);
        } else
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = f2h(d[k]);
        *at = o;
    }
    if (h.edge >= 0) to[h.edge] = combined(value(h.e) + (h.edge == x ? c : 0.f), a.acc, a.acc ? to[h.edge] : (half_t)0.f);
}

// gradient 0
template <int T, int NP>
__device__ __forceinline__ void put_nothing(const TokenArgs &a, half_t *to, const VocabRow &g, const Held<T, NP> &h)
{
    if (a.acc) return;
#pragma unroll
    for (int i = 0; i < NP; i++) {
        if (!h.has(i)) break;
        *reinterpret_cast<half8_t *>(to + g.first(h.piece(i))) = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
    }
    if (h.edge >= 0) to[h.edge] = (half_t)0.f;
}

template <int T, int NP>
__global__ void __launch_bounds__(T) logp_fwd_kernel(TokenArgs a)
{
    const int64_t n = blockIdx.x;
    const int x = token(a, n, threadIdx.x == 0);
    RowStats r = {0.f, 0.f, 0.f};              // (a sum of 0, which no row has: left out, and so by the adjoint)
    if (x >= 0) {
        const VocabRow z(a.logit + n * a.ld, a.V);
        Held<T, NP> h(z);
        h.load(z, z);
        r = row_stats(h, h2f(z.row[x]), a.inv_temp);
    }
    if (threadIdx.x) return;
    a.logp[n] = r.logp;
    a.stats[2 * n] = r.mx;
    a.stats[2 * n + 1] = r.sum;
}

template <int T, int NP>
__global__ void __launch_bounds__(T) logp_bwd_kernel(TokenArgs a)
{
    const int64_t n = blockIdx.x;
    const VocabRow z(a.logit + n * a.ld, a.V), g(a.grad + n * a.ldd, a.V);
    half_t *to = a.grad + n * a.ldd;
    Held<T, NP> h(g);
    const float d = a.dlogp[n], mx = a.stats[2 * n], sum = a.stats[2 * n + 1];
    const int x = a.tok[n];
    if (d == 0.f || sum == 0.f || x >= a.V) return put_nothing(a, to, g, h);
    h.load(z, g);
    put_gradient(a, to, g, h, x, mx, sum, d * a.inv_temp);
}

// e^d - 1 - d, also where d is small and the difference would cancel
__device__ __forceinline__ float exp_beyond_line(float d)
{
    if (!(fabsf(d) <= 0.5f)) return expm1f(d) - d;
    // d^2 (1/2! + d/3! + .. + d^7/9!), the next term below 2^-25 of it
    float s = 1.f / 362880;
    s = s * d + 1.f / 40320;
    s = s * d + 1.f / 5040;
    s = s * d + 1.f / 720;
    s = s * d + 1.f / 120;
    s = s * d + 1.f / 24;
    s = s * d + 1.f / 6;
    s = s * d + 0.5f;
    return s * d * d;
}

// a e^x, also where only e^x is beyond fp32 (e^64 = kFar is taken out of it first, exactly where it matters); of a = 0 nothing, unless x is no number
constexpr float kFar = 6.2351490808116169e27f;
__device__ __forceinline__ float times_exp(float a, float x)
{
    if (a == 0.f && x == x) return a;
    const bool far = x > 64.f;
    const float e = a * expf(far ? x - 64.f : x);
    return far ? e * kFar : e;
}

template <int T, int NP>
__global__ void __launch_bounds__(T) policy_kernel(TokenArgs a)
{
    const int64_t n = blockIdx.x;
    const VocabRow z(a.logit + n * a.ld, a.V), g(a.grad + n * a.ldd, a.V);
    half_t *to = a.grad + n * a.ldd;
    Held<T, NP> h(g);
    const int x = token(a, n, threadIdx.x == 0);
    if (x < 0) {
        if (threadIdx.x == 0) a.loss[n] = a.logp[n] = 0.f;
        return put_nothing(a, to, g, h);
    }
    h.load(z, g);
    const float zx = h2f(z.row[x]), old = a.old[n], adv = a.adv[n], ref = a.ref ? a.ref[n] : 0.f, scale = a.scale[n];
    const RowStats r = row_stats(h, zx, a.inv_temp);
    const float ratio = expf(r.logp - old), clipped = fminf(fmaxf(ratio, 1.f - a.lo), 1.f + a.hi);
    const float free = times_exp(adv, r.logp - old), bound = clipped * adv;
    // (a NaN in either stays one)
    float loss = free <= bound ? -free : free > bound ? -bound : NAN;
    float slope = free <= bound ? -free : free > bound ? 0.f : NAN;
    if (a.ref && a.beta > 0.f) {
        const float d = ref - r.logp;
        const bool far = d > 64.f;             // (1 and d are below 2^-80 of e^d)
        loss += far ? times_exp(a.beta, d) : a.beta * exp_beyond_line(d);
        slope -= far ? times_exp(a.beta, d) : a.beta * expm1f(d);
    }
    if (threadIdx.x == 0) {
        a.loss[n] = loss;
        a.logp[n] = r.logp;
    }
    const float c = scale == 0.f && slope == slope ? 0.f : slope * scale * a.inv_temp;       // (none of an infinite slope is nothing)
    if (c == 0.f) return put_nothing(a, to, g, h);
    put_gradient(a, to, g, h, x, r.mx, r.sum, c);
}

// Threads and pieces that hold a row: one wave to a short one (300 wide, 437000 rows: the policy loss 269 us, by 256 threads 727), as few pieces
// as do above 8199 (8200 wide, 16000 rows, log-probabilities: 44 us, with 512 threads 62), else what measured 5.2 to 5.6 TB/s; above 32775
// 16 pieces, whose exponentials are not held beside them (92 registers; 50257 wide 104 us, with them in 160 132).
#define CACTI_BY_WIDTH(kernel, a, st)                                                                            \
    do {                                                                                                         \
        const dim3 grid((unsigned)(a).N);                                                                        \
        if ((a).V < 8 * 64 * 4 + 8) hipLaunchKernelGGL((kernel<64, 4>), grid, dim3(64), 0, st, a);               \
        else if ((a).V < 8 * 256 * 4 + 8) hipLaunchKernelGGL((kernel<256, 4>), grid, dim3(256), 0, st, a);       \
        else if ((a).V < 8 * 256 * 5 + 8) hipLaunchKernelGGL((kernel<256, 5>), grid, dim3(256), 0, st, a);       \
        else if ((a).V < 8 * 512 * 4 + 8) hipLaunchKernelGGL((kernel<512, 4>), grid, dim3(512), 0, st, a);       \
        else if ((a).V < 8 * 512 * 8 + 8) hipLaunchKernelGGL((kernel<512, 8>), grid, dim3(512), 0, st, a);       \
        else hipLaunchKernelGGL((kernel<512, 16>), grid, dim3(512), 0, st, a);                                   \
    } while (0)

int check(const char *who, int64_t N, int64_t V, const void *logit, int64_t ld, const void *tok, double temperature, const void *status, TokenArgs *a)
{
    CACTI_REQUIRE(N > 0 && V > 0, CACTI_E_INVALID, "%s: empty shape", who);
    CACTI_REQUIRE(logit && tok, CACTI_E_INVALID, "%s: null pointer", who);
    CACTI_REQUIRE(V <= 65536 && N < (1 << 23), CACTI_E_NOTIMPL, "%s: at most 65536 tokens, 2^23 rows", who);
    CACTI_REQUIRE(ld >= V, CACTI_E_INVALID, "%s: row pitch below a row", who);
    CACTI_REQUIRE(temperature >= 1e-6 && temperature <= 1e6, CACTI_E_INVALID, "%s: temperature out of range", who);
    CACTI_REQUIRE(aligned(logit, 2) && aligned(tok, 2) && aligned(status, 4), CACTI_E_INVALID, "%s: misaligned operand", who);
    *a = TokenArgs{};
    a->N = N;
    a->V = (int)V;
    a->logit = (const half_t *)logit;
    a->ld = ld;
    a->tok = (const uint16_t *)tok;
    a->inv_temp = (float)(1. / temperature);
    a->status = (int *)const_cast<void *>(status);
    return 0;
}

int check_gradient(const char *who, void *dlogit16, int64_t ldd, int acc, TokenArgs *a)
{
    CACTI_REQUIRE(dlogit16 && aligned(dlogit16, 2), CACTI_E_INVALID, "%s: gradient null or misaligned", who);
    CACTI_REQUIRE(ldd >= a->V, CACTI_E_INVALID, "%s: row pitch below a row", who);
    // in place: a workgroup has read its row before it writes one
    CACTI_REQUIRE((a->logit == dlogit16 && (a->ld == ldd || a->N == 1)) || !rows_share(a->N, a->logit, a->ld, a->V, dlogit16, ldd, a->V), CACTI_E_INVALID,
                  "%s: the gradient takes the logits' place, with the same pitch, or shares no memory with them", who);
    a->grad = (half_t *)dlogit16;
    a->ldd = ldd;
    a->acc = acc;
    return 0;
}

// ---------------------------------------------------------------- pairs
struct PairArgs {
    int64_t N;
    int pairs;
    const float *logp, *ref, *scale;
    const int *starts;
    const uint8_t *mask;
    double beta, eps;
    int mean;
    float *loss, *reward, *dlogp;
    int *status;
};

constexpr int kPairThreads = 256;

__device__ __forceinline__ double block_sum_f64(double v, double *red)
{
    v = wave_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.;
#pragma unroll
    for (int w = 0; w < kPairThreads / 64; w++) v += red[w];
    return v;
}

__device__ __forceinline__ double log_sigmoid(double x) { return fmin(x, 0.) - log1p(exp(-fabs(x))); }

// Whether the rows of pair i are there
__device__ __forceinline__ bool there(const PairArgs &a, int i)
{
    const int *s = a.starts + 2 * i;
    return s[0] >= 0 && s[1] >= s[0] && s[2] >= s[1] && s[2] <= a.N;
}

// A workgroup to a pair, and one for the rows before the first and behind the last.  Where pairs are not there the first of a run of them clears what
// lies between those on either side that are: a number that is wrong says nothing of where other pairs' rows are.
__global__ void __launch_bounds__(kPairThreads) preference_kernel(PairArgs a)
{
    __shared__ double red[kPairThreads / 64];
    __shared__ int next;
    const int i = blockIdx.x, N = (int)a.N;
    auto clear = [&](int first, int last) __attribute__((always_inline)) {
        for (int n = first + (int)threadIdx.x; n < last; n += kPairThreads) a.dlogp[n] = 0.f;
    };
    if (i == a.pairs) {
        if (there(a, 0)) clear(0, a.starts[0]);
        if (there(a, a.pairs - 1)) clear(a.starts[2 * a.pairs], N);
        return;
    }
    const int s[3] = {a.starts[2 * i], a.starts[2 * i + 1], a.starts[2 * i + 2]};
    if (!there(a, i)) {
        if (threadIdx.x == 0) {
            a.loss[i] = a.reward[2 * i] = a.reward[2 * i + 1] = 0.f;
            if (a.status) atomicMax(a.status, i + 1);
            next = a.pairs;
        }
        if (i > 0 && !there(a, i - 1)) return;
        __syncthreads();
        for (int j = i + 1 + (int)threadIdx.x; j < a.pairs; j += kPairThreads)
            if (there(a, j)) {
                atomicMin(&next, j);
                break;
            }
        __syncthreads();
        clear(i > 0 ? s[0] : 0, next < a.pairs ? a.starts[2 * next] : N);
        return;
    }
    double reward[2], each[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        double sum = 0.;
        int count = 0;
        for (int n = s[t] + (int)threadIdx.x; n < s[t + 1]; n += kPairThreads) {
            if (a.mask && !a.mask[n]) continue;
            sum += (double)a.logp[n] - (a.ref ? (double)a.ref[n] : 0.);
            count++;
        }
        sum = block_sum_f64(sum, red);
        each[t] = a.beta;
        if (a.mean) each[t] /= fmax(block_sum_f64((double)count, red), 1.);
        reward[t] = each[t] * sum;
    }
    const double h = reward[0] - reward[1];
    const double slope = a.scale[i] * (a.eps / (1. + exp(-h)) - (1. - a.eps) / (1. + exp(h)));
    if (threadIdx.x == 0) {
        // (a share of 0 of an infinite loss is none)
        a.loss[i] = (float)((a.eps < 1. ? -(1. - a.eps) * log_sigmoid(h) : 0.) - (a.eps > 0. ? a.eps * log_sigmoid(-h) : 0.));
        a.reward[2 * i] = (float)reward[0];
        a.reward[2 * i + 1] = (float)reward[1];
    }
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const float d = (float)((t ? -slope : slope) * each[t]);
        for (int n = s[t] + (int)threadIdx.x; n < s[t + 1]; n += kPairThreads) a.dlogp[n] = a.mask && !a.mask[n] ? 0.f : d;
    }
}

}  // namespace

CACTI_API int cacti_hip_token_logp_fwd(int64_t N, int64_t V, const void *logit16, int64_t ld, const void *tok, const void *mask,
                                       double temperature, void *logp, void *stats, void *status, void *stream)
{
    TokenArgs a;
    const int rc = check("token_logp_fwd", N, V, logit16, ld, tok, temperature, status, &a);
    if (rc) return rc;
    CACTI_REQUIRE(logp && stats && aligned(logp, 4) && aligned(stats, 4), CACTI_E_INVALID, "token_logp_fwd: logp or stats null or misaligned");
    a.mask = (const uint8_t *)mask;
    a.logp = (float *)logp;
    a.stats = (float *)stats;
    CACTI_BY_WIDTH(logp_fwd_kernel, a, (hipStream_t)stream);
    return launch_status("token_logp_fwd");
}

CACTI_API int cacti_hip_token_logp_bwd(int64_t N, int64_t V, const void *logit16, int64_t ld, const void *tok, const void *stats,
                                       const void *dlogp, double temperature, void *dlogit16, int64_t ldd, int acc, void *stream)
{
    TokenArgs a;
    int rc = check("token_logp_bwd", N, V, logit16, ld, tok, temperature, nullptr, &a);
    if (!rc) rc = check_gradient("token_logp_bwd", dlogit16, ldd, acc, &a);
    if (rc) return rc;
    CACTI_REQUIRE(stats && dlogp && aligned(stats, 4) && aligned(dlogp, 4), CACTI_E_INVALID, "token_logp_bwd: stats or dlogp null or misaligned");
    a.stats = (float *)const_cast<void *>(stats);
    a.dlogp = (const float *)dlogp;
    CACTI_BY_WIDTH(logp_bwd_kernel, a, (hipStream_t)stream);
    return launch_status("token_logp_bwd");
}

CACTI_API int cacti_hip_policy_loss(int64_t N, int64_t V, const void *logit16, int64_t ld, const void *tok, const void *mask, const void *old,
                                    const void *adv, const void *ref, const void *scale, double clip_lo, double clip_hi, double beta,
                                    double temperature, void *loss, void *logp, void *dlogit16, int64_t ldd, int acc, void *status, void *stream)
{
    TokenArgs a;
    int rc = check("policy_loss", N, V, logit16, ld, tok, temperature, status, &a);
    if (!rc) rc = check_gradient("policy_loss", dlogit16, ldd, acc, &a);
    if (rc) return rc;
    CACTI_REQUIRE(old && adv && scale && loss && logp, CACTI_E_INVALID, "policy_loss: null pointer");
    CACTI_REQUIRE(aligned(old, 4) && aligned(adv, 4) && aligned(ref, 4) && aligned(scale, 4) && aligned(loss, 4) && aligned(logp, 4), CACTI_E_INVALID,
                  "policy_loss: misaligned operand");
    CACTI_REQUIRE(clip_lo >= 0. && clip_lo <= 1. && clip_hi >= 0. && clip_hi <= 1e6, CACTI_E_INVALID, "policy_loss: clip out of range");
    CACTI_REQUIRE(beta >= 0. && beta <= 1e6, CACTI_E_INVALID, "policy_loss: beta out of range");
    a.mask = (const uint8_t *)mask;
    a.old = (const float *)old;
    a.adv = (const float *)adv;
    a.ref = (const float *)ref;
    a.scale = (const float *)scale;
    a.lo = (float)clip_lo;
    a.hi = (float)clip_hi;
    a.beta = (float)beta;
    a.loss = (float *)loss;
    a.logp = (float *)logp;
    CACTI_BY_WIDTH(policy_kernel, a, (hipStream_t)stream);
    return launch_status("policy_loss");
}

CACTI_API int cacti_hip_preference_loss(int64_t N, int64_t pairs, const void *logp, const void *ref, const void *mask, const void *starts,
                                        const void *scale, double beta, double smoothing, int mean, void *loss, void *reward, void *dlogp,
                                        void *status, void *stream)
{
    CACTI_REQUIRE(N > 0 && pairs > 0, CACTI_E_INVALID, "preference_loss: empty shape");
    CACTI_REQUIRE(N < (1 << 23) && pairs < (1 << 23), CACTI_E_NOTIMPL, "preference_loss: at most 2^23 rows and pairs");
    CACTI_REQUIRE(logp && starts && scale && loss && reward && dlogp, CACTI_E_INVALID, "preference_loss: null pointer");
    CACTI_REQUIRE(aligned(logp, 4) && aligned(ref, 4) && aligned(starts, 4) && aligned(scale, 4) && aligned(loss, 4) && aligned(reward, 4) &&
                      aligned(dlogp, 4) && aligned(status, 4),
                  CACTI_E_INVALID, "preference_loss: misaligned operand");
    CACTI_REQUIRE(beta >= 0. && beta <= 1e6, CACTI_E_INVALID, "preference_loss: beta out of range");
    CACTI_REQUIRE(smoothing >= 0. && smoothing <= 1., CACTI_E_INVALID, "preference_loss: smoothing out of range");
    const PairArgs a = {N, (int)pairs, (const float *)logp, (const float *)ref, (const float *)scale, (const int *)starts, (const uint8_t *)mask,
                        beta, smoothing, mean, (float *)loss, (float *)reward, (float *)dlogp, (int *)status};
    hipLaunchKernelGGL(preference_kernel, dim3((unsigned)pairs + 1), dim3(kPairThreads), 0, (hipStream_t)stream, a);
    return launch_status("preference_loss");
}
