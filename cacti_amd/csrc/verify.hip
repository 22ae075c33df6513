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
//
// A workgroup per row: maxima, sums, whether the drafted token is kept and, unless it is, the token that would follow; then a
// workgroup per sequence picks the first row that ends it.
#include "vocab_row.h"

using namespace cacti;

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

struct VerifyArgs {
    int T, B, V;
    const half_t *target, *draft;
    int64_t ldt, ldd;
    const uint16_t *tok;
    const int *starts;
    const float *u, *r;
    double inv_temp;                           // 0: greedy
    int *verdict;                              // [T]: -1 where the drafted token is kept, else the token that follows the row
    int *accepted;
    uint16_t *next;
    int *status;
};

// A NaN is never chosen; the difference of equal infinities is 0
__device__ __forceinline__ float clean(half_t x) { return x != x ? -INFINITY : h2f(x); }
__device__ __forceinline__ double weight(float x, float mx, double inv_temp)
{
    return x == mx ? 1.0 : x == -INFINITY ? 0.0 : exp(((double)x - (double)mx) * inv_temp);
}

__device__ double block_sum(double v, double *red)
{
    v = wave_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.;
    for (int w = 0; w < kWaves; w++) s += red[w];
    return s;
}

// The sequence of a row, or B: starts do not fall
__device__ int sequence_of(const VerifyArgs &a, int row)
{
    int c = 0;
    for (int i0 = 1; i0 <= a.B; i0 += 64) {
        const int i = i0 + (threadIdx.x & 63);
        c += __popcll(__ballot(i <= a.B && a.starts[i] <= row));
    }
    return c;
}

__global__ void __launch_bounds__(kThreads) verify_rows_kernel(VerifyArgs a)
{
    __shared__ float red[kWaves];
    __shared__ double redd[kWaves];
    __shared__ unsigned found;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int b = sequence_of(a, row);
    if (b >= a.B || row < a.starts[b]) return;
    const bool last = row + 1 >= a.starts[b + 1] || row + 1 >= a.T;
    const int x = last ? -1 : a.tok[row + 1];
    const bool bad = !last && x >= a.V;        // never kept
    if (bad && tid == 0 && a.status) atomicMax(a.status, row + 2);
    const VocabRow t(a.target + row * a.ldt, a.V);
    const bool greedy = a.inv_temp == 0.;
    const bool drafted = a.draft && !last && !greedy;
    const VocabRow d(drafted ? a.draft + row * a.ldd : t.row, a.V);
    float mt = -INFINITY, md = -INFINITY;
    for (int c = tid; c < t.pieces(); c += kThreads) {
        const h8 v = t.load(c, (half_t)-INFINITY);
#pragma unroll
        for (int k = 0; k < 8; k++) mt = fmaxf(mt, clean(v.v[k]));
    }
    mt = block_reduce(mt, OpMax(), -INFINITY, red);
    if (greedy) {
        if (tid == 0) found = 0xffffffffu;
        __syncthreads();
        for (int c = tid; c < t.pieces(); c += kThreads) {
            const h8 v = t.load(c, (half_t)-INFINITY);
#pragma unroll
            for (int k = 7; k >= 0; k--) {
                const int j = t.first(c) + k;
                if (j >= 0 && j < a.V && clean(v.v[k]) == mt) atomicMin(&found, (unsigned)j);
            }
        }
        __syncthreads();
        if (tid == 0) a.verdict[row] = !last && !bad && x == (int)found && a.u[row] < 1.f ? -1 : (int)found;
        return;
    }
    double zt = 0., zd = 1.;
    for (int c = tid; c < t.pieces(); c += kThreads) {
        const h8 v = t.load(c, (half_t)-INFINITY);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int j = t.first(c) + k;
            if (j >= 0 && j < a.V) zt += weight(clean(v.v[k]), mt, a.inv_temp);
        }
    }
    zt = block_sum(zt, redd);
    if (drafted) {
        for (int c = tid; c < d.pieces(); c += kThreads) {
            const h8 v = d.load(c, (half_t)-INFINITY);
#pragma unroll
            for (int k = 0; k < 8; k++) md = fmaxf(md, clean(v.v[k]));
        }
        md = block_reduce(md, OpMax(), -INFINITY, red);
        zd = 0.;
        for (int c = tid; c < d.pieces(); c += kThreads) {
            const h8 v = d.load(c, (half_t)-INFINITY);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int j = d.first(c) + k;
                if (j >= 0 && j < a.V) zd += weight(clean(v.v[k]), md, a.inv_temp);
            }
        }
        zd = block_sum(zd, redd);
    }
    const double it = 1. / zt, id = 1. / zd;
    if (!last && !bad) {
        const double p = weight(clean(t.row[x]), mt, a.inv_temp) * it;
        const double q = drafted ? weight(clean(d.row[x]), md, a.inv_temp) * id : 1.;
        if ((double)a.u[row] * q < p) {
            if (tid == 0) a.verdict[row] = -1;
            return;
        }
    }
    // weight of token j of what is left; residual: what the drafting model does not have of it
    auto left = [&](int j, bool residual) {
        double w = weight(clean(t.row[j]), mt, a.inv_temp) * it;
        if (residual) w = drafted ? w - weight(clean(d.row[j]), md, a.inv_temp) * id : j == x ? 0. : w;
        return w > 0. ? w : 0.;
    };
    // a lane has a run of tokens, lanes and waves those that follow
    const int per = (a.V + kThreads - 1) / kThreads, j0 = min(tid * per, a.V), j1 = min(j0 + per, a.V);
    bool residual = !last;
    double mine = 0., total;
    for (;;) {
        mine = 0.;
        for (int j = j0; j < j1; j++) mine += left(j, residual);
        total = block_sum(mine, redd);
        if (total > 0. || !residual) break;
        residual = false;                      // p = q: nothing is left of it
    }
    const double want = (double)a.r[b] * total;
    double before = 0.;                        // of the waves before this one
    for (int w = 0; w < wid; w++) before += redd[w];
    double upto = mine;                        // inclusive sum over the lanes
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const double o = __shfl_up(upto, s);
        if (lane >= s) upto += o;
    }
    upto += before;
    if (tid == 0) found = 0xffffffffu;
    __syncthreads();
    if (upto > want && mine > 0.) atomicMin(&found, (unsigned)tid);
    __syncthreads();
    unsigned owner = found;
    if (owner == 0xffffffffu) {                // beyond the last by a rounding: the last with any weight
        __syncthreads();
        if (tid == 0) found = 0;
        __syncthreads();
        if (mine > 0.) atomicMax(&found, (unsigned)tid);
        __syncthreads();
        owner = found;
    }
    if (tid == (int)owner) {
        double c = upto - mine;
        int pick = j0;
        for (int j = j0; j < j1; j++) {
            const double w = left(j, residual);
            c += w;
            if (w > 0.) pick = j;
            if (w > 0. && c > want) break;
        }
        a.verdict[row] = min(pick, a.V - 1);
    }
}

__global__ void __launch_bounds__(64) verify_pick_kernel(VerifyArgs a)
{
    const int b = blockIdx.x, lane = threadIdx.x;
    const int s0 = a.starts[b], s1 = a.starts[b + 1];
    if (s0 < 0 || s1 > a.T || s1 < s0) {
        if (lane == 0 && a.status) atomicMax(a.status, 1);
        if (lane == 0) a.accepted[b] = 0;
        return;
    }
    int end = s1;                              // the first row that is not kept
    for (int i0 = s0; i0 < s1 && end == s1; i0 += 64) {
        const uint64_t stop = __ballot(i0 + lane < s1 && a.verdict[min(i0 + lane, s1 - 1)] >= 0);
        if (stop) end = i0 + __ffsll((unsigned long long)stop) - 1;
    }
    for (int i = s0 + lane; i < s1; i += 64) a.next[i] = i < end ? a.tok[min(i + 1, a.T - 1)] : i == end ? (uint16_t)a.verdict[i] : (uint16_t)0;
    if (lane == 0) a.accepted[b] = s1 > s0 ? end - s0 : 0;
}

}  // namespace

CACTI_API size_t cacti_hip_verify_draft_workspace(int64_t T, int64_t V)
{
    return T > 0 && V > 0 ? (size_t)T * 4 : 0;
}

CACTI_API int cacti_hip_verify_draft_f16(int64_t T, int64_t B, int64_t V, const void *target, int64_t ldt, const void *draft, int64_t ldd,
                                         const void *tok, const void *starts, const void *u, const void *r, double temperature, void *accepted,
                                         void *next, void *workspace, size_t workspace_bytes, void *status, void *stream)
{
    CACTI_REQUIRE(T > 0 && B > 0 && V > 0, CACTI_E_INVALID, "verify_draft: empty shape");
    CACTI_REQUIRE(target && tok && starts && u && r && accepted && next && workspace, CACTI_E_INVALID, "verify_draft: null pointer");
    CACTI_REQUIRE(V <= 65536 && T < (1 << 22) && B <= (1 << 22), CACTI_E_NOTIMPL, "verify_draft: at most 65536 tokens and 2^22 rows");
    CACTI_REQUIRE(ldt >= V && (!draft || ldd >= V), CACTI_E_INVALID, "verify_draft: row pitch below a row");
    CACTI_REQUIRE(temperature >= 0. && temperature <= 1e30 && (temperature == 0. || temperature >= 1e-30), CACTI_E_INVALID,
                  "verify_draft: the temperature is 0 or positive");
    CACTI_REQUIRE(aligned(target, 2) && aligned(draft, 2) && aligned(tok, 2) && aligned(next, 2) && aligned(starts, 4) && aligned(u, 4) &&
                      aligned(r, 4) && aligned(accepted, 4) && aligned(workspace, 4) && aligned(status, 4),
                  CACTI_E_INVALID, "verify_draft: misaligned operand");
    CACTI_REQUIRE(workspace_bytes >= cacti_hip_verify_draft_workspace(T, V), CACTI_E_INVALID, "verify_draft: workspace too small");
    const VerifyArgs a = {(int)T, (int)B, (int)V, (const half_t *)target, (const half_t *)draft, ldt, ldd, (const uint16_t *)tok,
                          (const int *)starts, (const float *)u, (const float *)r, temperature == 0. ? 0. : 1. / temperature,
                          (int *)workspace, (int *)accepted, (uint16_t *)next, (int *)status};
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)T), dim3(kThreads), 0, st, a);
    const int rc = launch_status("verify_draft");
    if (rc) return rc;
    hipLaunchKernelGGL(verify_pick_kernel, dim3((unsigned)B), dim3(64), 0, st, a);
    return launch_status("verify_draft (pick)");
}
