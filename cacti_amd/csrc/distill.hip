// Distillation from a teacher's top logits: per row K token ids idx and the teacher's logits val of them, against the student's
// logits z over the vocabulary, both at a temperature tau:
//   t = softmax(val / tau),  p = softmax(z / tau)
//   loss = sum_i t_i (log t_i - log p(idx_i))
//   dz_j = scale / tau (p_j sum(t) - sum_{i: idx_i = j} t_i)
// An entry of -inf has no weight (padding); a row of none but such has loss 0 and gradient 0.
//
// A workgroup to a row, which it holds in registers from one read on: the forward pass is bound by that read, the adjoint, which
// takes the maximum and the sum from the forward pass (stats) and has nothing to reduce over the row, by a read and a write.
// 2048 rows of 32000, K = 64, each call after calls of its kind: forward 26 us, 5.0 TB/s (a maximum and then a sum out of memory again:
// 44), adjoint 47 us, 5.6 TB/s, and one after the other, when the forward pass has the gradients written before it go to memory beside
// it, 86; 611 of 8191, K = 20: 5.8 and 6.7 us; 128 of 1024, K = 8: 4.2 and 3.9 us, latency.
#include "operands.h"
#include "vocab_row.h"

using namespace cacti;

namespace {

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

// The teacher's entries of a thread: tid, tid + T, ...
template <int T>
struct Entries {
    static constexpr int kOf = kMaxK / T;
    half_t v[kOf], z[kOf];                     // the teacher's logit (-inf behind the last) and the student's
    int j[kOf];
    __device__ __forceinline__ void load(const DistillArgs &a, int64_t n, const half_t *row)
    {
#pragma unroll
        for (int e = 0; e < kOf; e++) {
            v[e] = z[e] = (half_t)-INFINITY;
            j[e] = a.V;
            if (e > 0 && e * T >= a.K) continue;
            const int i = (int)threadIdx.x + e * T, ic = min(i, a.K - 1);
            const half_t x = a.val[n * a.K + ic];
            j[e] = a.idx[n * a.K + ic];
            z[e] = row[min(j[e], a.V - 1)];
            v[e] = i < a.K ? x : (half_t)-INFINITY;
            j[e] = i < a.K ? j[e] : -1;
        }
    }
    __device__ __forceinline__ float max() const
    {
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < kOf; e++) m = fmaxf(m, h2f(v[e]));
        return m;
    }
    // e^((v - mx) / tau); mx = -inf: there is none but -inf and NaN
    __device__ __forceinline__ float weight(int e, float mx, double inv_temp) const
    {
        if (mx == -INFINITY) return v[e] != v[e] ? NAN : 0.f;
        return expf((float)(((double)h2f(v[e]) - (double)mx) * inv_temp));
    }
};

template <int T>
__device__ __forceinline__ void block_max2(float &x, float &y)
{
    __shared__ float red[T / 64][2];
    x = wave_reduce(x, OpMax());
    y = wave_reduce(y, OpMax());
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6][0] = x;
        red[threadIdx.x >> 6][1] = y;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        x = fmaxf(x, red[w][0]);
        y = fmaxf(y, red[w][1]);
    }
}

template <int T, int NP>
__global__ void __launch_bounds__(T) distill_fwd_kernel(DistillArgs a)
{
    __shared__ float sums[T / 64][3];
    __shared__ double parts[T / 64];
    const int64_t n = blockIdx.x;
    const VocabRow z(a.logit + n * a.ld, a.V);
    Entries<T> t;
    Held<T, NP> h(z);
    t.load(a, n, z.row);
    h.load(z, z);
    const float c2 = (float)(a.inv_temp * 1.44269504088896340736);
    if (h.edge < 0) h.e = (half_t)-INFINITY;
    float mx = h2f(h.e), tmx = t.max();
    if (h.hi > h.lo) {                         // (what a thread does not have is some other element of the row)
        half8_t m8 = h.x[0];
#pragma unroll
        for (int i = 1; i < NP; i++) m8 = __builtin_elementwise_max(m8, h.x[i]);
#pragma unroll
        for (int k = 0; k < 8; k++) mx = fmaxf(mx, h2f(m8[k]));
    }
    block_max2<T>(mx, tmx);
    float s = __builtin_amdgcn_exp2f((h2f(h.e) - mx) * c2);
    s = h.edge < 0 ? 0.f : s;
#pragma unroll
    for (int i = 0; i < NP; i++) {
        float p = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) p += __builtin_amdgcn_exp2f((h2f(h.x[i][k]) - mx) * c2);
        s += h.has(i) ? p : 0.f;
    }
    // log t_i - log p_i = ((val_i - val_max) - (z_i - z_max)) / tau + log(sum_z / sum_t)
    float sum = 0.f, valid = 0.f;
    double part = 0.;
#pragma unroll
    for (int e = 0; e < Entries<T>::kOf; e++) {
        if (e * T >= a.K) break;
        const float w = t.weight(e, tmx, a.inv_temp);
        sum += w;
        if (t.j[e] >= a.V && a.status) atomicMax(a.status, (int)min(n + 1, (int64_t)INT32_MAX));
        if (t.j[e] >= a.V || w == 0.f) continue;
        valid += w;
        part += (double)w * (((double)h2f(t.v[e]) - (double)tmx) * a.inv_temp - ((double)h2f(t.z[e]) - (double)mx) * a.inv_temp);
    }
    s = wave_sum(s);
    sum = wave_sum(sum);
    valid = wave_sum(valid);
    part = wave_sum_f64(part);
    if ((threadIdx.x & 63) == 0) {
        const int w = threadIdx.x >> 6;
        sums[w][0] = s;
        sums[w][1] = sum;
        sums[w][2] = valid;
        parts[w] = part;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = sum = valid = 0.f;
        part = 0.;
#pragma unroll
        for (int w = 0; w < T / 64; w++) {
            s += sums[w][0];
            sum += sums[w][1];
            valid += sums[w][2];
            part += parts[w];
        }
        a.loss[n] = valid == 0.f && sum == sum ? 0.f : (float)((part + (double)valid * (log((double)s) - log((double)sum))) / (double)sum);
        a.stats[2 * n] = mx;
        a.stats[2 * n + 1] = s;
    }
}

template <int T, int NP>
__global__ void __launch_bounds__(T) distill_bwd_kernel(DistillArgs a)
{
    constexpr int kOf = Entries<T>::kOf;
    __shared__ float sums[T / 64][2];
    __shared__ __attribute__((aligned(16))) int ids[kMaxK];
    __shared__ __attribute__((aligned(16))) float es[kMaxK];
    const int64_t n = blockIdx.x;
    const VocabRow z(a.logit + n * a.ld, a.V), g(a.grad + n * a.ldd, a.V);
    half_t *gr = a.grad + n * a.ldd;
    Entries<T> t;
    Held<T, NP> h(g);                          // the gradient's pieces
    t.load(a, n, z.row);
    const float mx = a.stats[2 * n], row_sum = a.stats[2 * n + 1], scale = a.scale[n];
    // all that is read of the logits and, of other threads' pieces, of the gradient is read before anything is written
    h.load(z, g);
    half_t old[kOf];
#pragma unroll
    for (int e = 0; e < kOf; e++) {
        old[e] = (half_t)0.f;
        if (a.acc && e * T < a.K) old[e] = gr[min(max(t.j[e], 0), a.V - 1)];
    }
    float tmx = t.max(), none = 0.f;
    block_max2<T>(tmx, none);
    float sum = 0.f, valid = 0.f;
#pragma unroll
    for (int e = 0; e < kOf; e++) {
        if (e * T >= a.K) break;
        const float w = t.weight(e, tmx, a.inv_temp);
        sum += w;
        if (t.j[e] < a.V) valid += w;
        ids[threadIdx.x + e * T] = t.j[e];     // (-1 behind the last)
        es[threadIdx.x + e * T] = w;
    }
    sum = wave_sum(sum);
    valid = wave_sum(valid);
    if ((threadIdx.x & 63) == 0) {
        sums[threadIdx.x >> 6][0] = sum;
        sums[threadIdx.x >> 6][1] = valid;
    }
    __syncthreads();
    sum = valid = 0.f;
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        sum += sums[w][0];
        valid += sums[w][1];
    }
    const bool empty = valid == 0.f && sum == sum;
    const float c2 = (float)(a.inv_temp * 1.44269504088896340736), sc = (float)(scale * a.inv_temp), inv = valid / sum / row_sum;
    // (empty: a student's NaN must not meet the zero)
    auto stream = [&](half_t x) __attribute__((always_inline)) { return empty ? 0.f : sc * (__builtin_amdgcn_exp2f((h2f(x) - mx) * c2) * inv); };
    // the entries: the last of those with an id has them all, in order
    half_t entry[kOf];
    bool mine[kOf];
#pragma unroll
    for (int e = 0; e < kOf; e++) {
        const int i = (int)threadIdx.x + e * T, j = t.j[e];
        mine[e] = i < a.K && j < a.V;
        if (!mine[e]) continue;
        float w = 0.f;
        for (int k = 0; k < a.K; k += 4) {
            const int4 id = *reinterpret_cast<const int4 *>(ids + k);
            const float4 x = *reinterpret_cast<const float4 *>(es + k);
            w += id.x == j ? x.x : 0.f;
            w += id.y == j ? x.y : 0.f;
            w += id.z == j ? x.z : 0.f;
            w += id.w == j ? x.w : 0.f;
            const int last = id.w == j ? 3 : id.z == j ? 2 : id.y == j ? 1 : id.x == j ? 0 : -k;
            mine[e] = mine[e] && k + last <= i;
        }
        const float p = __builtin_amdgcn_exp2f((h2f(t.z[e]) - mx) * c2) * inv;
        entry[e] = combined(empty ? 0.f : sc * (p - w / sum), a.acc, old[e]);
    }
#pragma unroll
    for (int i = 0; i < NP; i++) {
        if (!h.has(i)) break;
        half_t *to = gr + g.first(h.piece(i));
        half8_t o;
        if (a.acc) {
            o = *reinterpret_cast<const half8_t *>(to);
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = combined(stream(h.x[i][k]), 1, o[k]);
        } else
#pragma unroll
            for (int k = 0; k < 8; k++) o[k] = f2h(stream(h.x[i][k]));
        *reinterpret_cast<half8_t *>(to) = o;
    }
    if (h.edge >= 0) gr[h.edge] = combined(stream(h.e), a.acc, a.acc ? gr[h.edge] : (half_t)0.f);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kOf; e++)
        if (mine[e]) gr[t.j[e]] = entry[e];
}

// The least threads and registers that hold a row.  (Forward and adjoint, 611 rows of 8191: 256 threads 5.8 and 6.7 us, 512 6.6 and
// 7.3; 2048 of 32000: 256 25.9 and 48.8, 512 26.1 and 47.0, 1024 32.6 and 58.6)
#define CACTI_DISTILL(kernel, a, st)                                                                                                  \
    do {                                                                                                                              \
        const dim3 grid((unsigned)(a).N);                                                                                             \
        if ((a).V < 8 * 256 * 4 + 8) hipLaunchKernelGGL((kernel<256, 4>), grid, dim3(256), 0, st, a);                                 \
        else if ((a).V < 8 * 512 * 4 + 8) hipLaunchKernelGGL((kernel<512, 4>), grid, dim3(512), 0, st, a);                            \
        else if ((a).V < 8 * 512 * 8 + 8) hipLaunchKernelGGL((kernel<512, 8>), grid, dim3(512), 0, st, a);                            \
        else hipLaunchKernelGGL((kernel<512, 16>), grid, dim3(512), 0, st, a);                                                        \
    } while (0)

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
    CACTI_DISTILL(distill_fwd_kernel, a, (hipStream_t)stream);
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
    // in place: a workgroup has read its row before it writes one
    CACTI_REQUIRE((logit16 == dlogit16 && (ld == ldd || N == 1)) || !rows_share(N, logit16, ld, V, dlogit16, ldd, V), CACTI_E_INVALID,
                  "distill_topk_bwd: the gradient takes the logits' place, with the same pitch, or shares no memory with them");
    a.scale = (const float *)scale;
    a.grad = (half_t *)dlogit16;
    a.ldd = ldd;
    a.acc = acc;
    CACTI_DISTILL(distill_bwd_kernel, a, (hipStream_t)stream);
    return launch_status("distill_topk_bwd");
}
