// Distillation from a teacher's top logits: per row K token ids idx and the teacher's logits val of them, against the student's
// logits z over the vocabulary, both at a temperature tau:
//   t = softmax(val / tau),  p = softmax(z / tau)
//   loss = sum_i t_i (log t_i - log p(idx_i))
//   dz_j = scale / tau (p_j sum(t) - sum_{i: idx_i = j} t_i)
// An entry of -inf has no weight (padding); a row of none but such has loss 0 and gradient 0.
//
// Forward: one pass for the maximum, one for the sum (out of L2).  It keeps both per row (stats), so that the gradient is a
// stream over the logits: nothing to reduce, one fma and one exponential per element.  The K entries are written again
// afterwards by the same workgroup, behind its barrier.
#include "vocab_row.h"

using namespace cacti;

namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMaxK = 1024;

struct DistillArgs {
    int64_t N;
    int V, K;
    const half_t *logit, *val;
    const uint16_t *idx;
    int64_t ld, ldd;
    double inv_temp;
    float *loss, *stats;
    const float *scale;
    half_t *grad;
    int acc;
    int *status;
};

// The teacher's K probabilities of a row by thread i (i, i + kThreads): max and sum of exponentials over the block
struct Teacher {
    float mx, sum;
};
__device__ __forceinline__ Teacher teacher(const DistillArgs &a, int64_t n, float *red)
{
    const half_t *v = a.val + n * a.K;
    Teacher t;
    float m = -INFINITY;
    bool nan = false;
    for (int i = threadIdx.x; i < a.K; i += kThreads) {
        m = fmaxf(m, h2f(v[i]));
        nan = nan || v[i] != v[i];
    }
    t.mx = block_reduce(m, OpMax(), -INFINITY, red);
    float s = 0.f;
    if (t.mx > -INFINITY)
        for (int i = threadIdx.x; i < a.K; i += kThreads) s += expf((float)(((double)h2f(v[i]) - (double)t.mx) * a.inv_temp));
    if (nan) s = NAN;
    t.sum = block_reduce(s, OpSum(), 0.f, red);
    return t;
}

__global__ void __launch_bounds__(kThreads) distill_fwd_kernel(DistillArgs a)
{
    __shared__ float red[kWaves];
    __shared__ double redd[kWaves];
    const int64_t n = blockIdx.x;
    const VocabRow z(a.logit + n * a.ld, a.V);
    const float c2 = (float)(a.inv_temp * 1.44269504088896340736);
    float mx = -INFINITY;
    for (int c = threadIdx.x; c < z.pieces(); c += kThreads) {
        const h8 v = z.load(c, (half_t)-INFINITY);
#pragma unroll
        for (int k = 0; k < 8; k++) mx = fmaxf(mx, h2f(v.v[k]));
    }
    mx = block_reduce(mx, OpMax(), -INFINITY, red);
    float s = 0.f;
    for (int c = threadIdx.x; c < z.pieces(); c += kThreads) {
        const h8 v = z.load(c, (half_t)-INFINITY);
#pragma unroll
        for (int k = 0; k < 8; k++) s += __builtin_amdgcn_exp2f((h2f(v.v[k]) - mx) * c2);
    }
    const float sum = block_reduce(s, OpSum(), 0.f, red);
    const Teacher t = teacher(a, n, red);
    // log t_i - log p_i = ((val_i - val_max) - (z_i - z_max)) / tau + log(sum_z / sum_t)
    const double shift = log((double)sum) - log((double)t.sum);
    double loss = 0.;
    for (int i = threadIdx.x; i < a.K; i += kThreads) {
        const int j = a.idx[n * a.K + i];
        if (j >= a.V) {
            if (a.status) atomicMax(a.status, (int)min(n + 1, (int64_t)INT32_MAX));
            continue;
        }
        const double dv = ((double)h2f(a.val[n * a.K + i]) - (double)t.mx) * a.inv_temp;
        const float w = expf((float)dv) / t.sum;
        if (w != 0.f) loss += (double)w * (dv - ((double)h2f(z.row[j]) - (double)mx) * a.inv_temp + shift);
    }
    loss = wave_sum_f64(loss);
    if ((threadIdx.x & 63) == 0) redd[threadIdx.x >> 6] = loss;
    __syncthreads();
    if (threadIdx.x == 0) {
        double l = 0.;
        for (int w = 0; w < kWaves; w++) l += redd[w];
        a.loss[n] = t.mx == -INFINITY && t.sum == 0.f ? 0.f : (float)l;
        a.stats[2 * n] = mx;
        a.stats[2 * n + 1] = sum;
    }
}

__device__ __forceinline__ half_t combined(float d, int acc, half_t old) { return acc ? f2h(h2f(old) + rnd16(d)) : f2h(d); }

__global__ void __launch_bounds__(kThreads) distill_bwd_kernel(DistillArgs a)
{
    __shared__ float red[kWaves];
    __shared__ uint16_t ids[kMaxK];
    __shared__ float ts[kMaxK];
    const int64_t n = blockIdx.x;
    const VocabRow z(a.logit + n * a.ld, a.V);
    half_t *gr = a.grad + n * a.ldd;
    const float c2 = (float)(a.inv_temp * 1.44269504088896340736), sc = (float)(a.scale[n] * a.inv_temp);
    const float mx = a.stats[2 * n], inv = 1.f / a.stats[2 * n + 1];
    const Teacher t = teacher(a, n, red);
    const bool empty = t.mx == -INFINITY && t.sum == 0.f;
    for (int i = threadIdx.x; i < a.K; i += kThreads) {
        const int j = a.idx[n * a.K + i];
        ids[i] = (uint16_t)j;
        ts[i] = j < a.V && !empty ? expf((float)(((double)h2f(a.val[n * a.K + i]) - (double)t.mx) * a.inv_temp)) / t.sum : 0.f;
    }
    __syncthreads();
    // the entries: the first of those with an id has them all, in order; what is there before is read before it is written over
    half_t entry[(kMaxK + kThreads - 1) / kThreads];
    int at[(kMaxK + kThreads - 1) / kThreads];
#pragma unroll
    for (int e = 0; e < (kMaxK + kThreads - 1) / kThreads; e++) {
        const int i = threadIdx.x + e * kThreads;
        at[e] = -1;
        if (i >= a.K || ids[i] >= a.V) continue;
        float w = 0.f;
        bool mine = true;
        for (int k = 0; k < a.K; k++)
            if (ids[k] == ids[i]) {
                mine = mine && k >= i;
                w += ts[k];
            }
        if (!mine) continue;
        at[e] = ids[i];
        const float p = empty ? 0.f : __builtin_amdgcn_exp2f((h2f(z.row[at[e]]) - mx) * c2) * inv;
        entry[e] = combined(empty ? 0.f : sc * (p - w), a.acc, a.acc ? gr[at[e]] : (half_t)0.f);
    }
    __syncthreads();
    const VocabRow g(gr, a.V);
    for (int c = threadIdx.x; c < g.pieces(); c += kThreads) {
        const int j0 = g.first(c);
        h8 v, o;
        if (g.whole(c) && z.off == g.off) v = ld8(z.row + j0);
        else
#pragma unroll
            for (int k = 0; k < 8; k++) v.v[k] = j0 + k >= 0 && j0 + k < a.V ? z.row[j0 + k] : (half_t)0.f;
        if (a.acc) o = g.load(c, (half_t)0.f);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float d = empty ? 0.f : sc * (__builtin_amdgcn_exp2f((h2f(v.v[k]) - mx) * c2) * inv);
            o.v[k] = combined(d, a.acc, o.v[k]);
        }
        if (g.whole(c)) st8(gr + j0, o);
        else
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (j0 + k >= 0 && j0 + k < a.V) gr[j0 + k] = o.v[k];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < (kMaxK + kThreads - 1) / kThreads; e++)
        if (at[e] >= 0) gr[at[e]] = entry[e];
}

int check(const char *who, int64_t N, int64_t V, int64_t K, const void *logit, int64_t ld, const void *idx, const void *val, const void *stats,
          double temperature, DistillArgs *a)
{
    CACTI_REQUIRE(N > 0 && V > 0 && K > 0, CACTI_E_INVALID, "%s: empty shape", who);
    CACTI_REQUIRE(logit && idx && val && stats, CACTI_E_INVALID, "%s: null pointer", who);
    CACTI_REQUIRE(V <= 65536 && K <= kMaxK && N < (1 << 23), CACTI_E_NOTIMPL, "%s: at most 65536 tokens, %d of them from the teacher, 2^23 rows",
                  who, kMaxK);
    CACTI_REQUIRE(ld >= V, CACTI_E_INVALID, "%s: row pitch below a row", who);
    CACTI_REQUIRE(temperature >= 1e-6 && temperature <= 1e6, CACTI_E_INVALID, "%s: temperature out of range", who);
    CACTI_REQUIRE(aligned(logit, 2) && aligned(idx, 2) && aligned(val, 2) && aligned(stats, 4), CACTI_E_INVALID, "%s: misaligned operand", who);
    *a = DistillArgs{N, (int)V, (int)K, (const half_t *)logit, (const half_t *)val, (const uint16_t *)idx, ld, 0, 1. / temperature,
                     nullptr, (float *)stats, nullptr, nullptr, 0, nullptr};
    return 0;
}

}  // namespace

CACTI_API int cacti_hip_distill_topk_fwd(int64_t N, int64_t V, int64_t K, const void *logit16, int64_t ld, const void *idx, const void *val16,
                                         double temperature, void *loss, void *stats, void *status, void *stream)
{
    DistillArgs a;
    const int rc = check("distill_topk_fwd", N, V, K, logit16, ld, idx, val16, stats, temperature, &a);
    if (rc) return rc;
    CACTI_REQUIRE(loss && aligned(loss, 4) && aligned(status, 4), CACTI_E_INVALID, "distill_topk_fwd: loss null or misaligned");
    a.loss = (float *)loss;
    a.status = (int *)status;
    hipLaunchKernelGGL(distill_fwd_kernel, dim3((unsigned)N), dim3(kThreads), 0, (hipStream_t)stream, a);
    return launch_status("distill_topk_fwd");
}

CACTI_API int cacti_hip_distill_topk_bwd(int64_t N, int64_t V, int64_t K, const void *logit16, int64_t ld, const void *idx, const void *val16,
                                         const void *stats, const void *scale, double temperature, void *dlogit16, int64_t ldd, int acc,
                                         void *stream)
{
    DistillArgs a;
    const int rc = check("distill_topk_bwd", N, V, K, logit16, ld, idx, val16, stats, temperature, &a);
    if (rc) return rc;
    CACTI_REQUIRE(scale && dlogit16 && aligned(scale, 4) && aligned(dlogit16, 2), CACTI_E_INVALID, "distill_topk_bwd: null pointer or misaligned operand");
    CACTI_REQUIRE(ldd >= V, CACTI_E_INVALID, "distill_topk_bwd: row pitch below a row");
    a.scale = (const float *)scale;
    a.grad = (half_t *)dlogit16;
    a.ldd = ldd;
    a.acc = acc;
    hipLaunchKernelGGL(distill_bwd_kernel, dim3((unsigned)N), dim3(kThreads), 0, (hipStream_t)stream, a);
    return launch_status("distill_topk_bwd");
}
