// Low-rank adapters of many requests beside a shared projection, and their gradients.  Row t of sequence s, with the adapter
// a = ids[s] (A_a [R, K], B_a [N, R], scale_a):
//   h = A_a x,  y = base + scale_a B_a h
//   dh = B_a^T dy,  dx = scale_a A_a^T dh,  dA_a = scale_a sum_t dh x^T,  dB_a = scale_a sum_t dy h^T   (over a's rows)
//
// All sums are fp32 (matrix instructions).  h and dh are one operand of a second product: they meet it as two f16 terms, value
// and what its rounding left, 22 bits in all, so that results are rounded once.  They are scaled by a power of two first, that of the
// largest of a row (for y and dx) or of the rows so far (for dA and dB): a gradient may lie far below f16's range and h beyond it.
// The terms lie side by side as 2 R columns, which for R = 16 fill the 32 that an instruction takes.
#include "operands.h"
#include "paged.h"

using namespace cacti;

namespace {

constexpr int kMaxR = 128;
constexpr int kTile = 16;                      // rows of a tile of h

struct AdapterArgs {
    PagedBatch pb;                             // T rows, sequences, starts, status
    Units units;
    int K, N, R, n, max_new;
    const half_t *x, *A, *B, *base;
    const int *ids;
    const float *scale;
    int64_t ldx, ldb, ldy;
    half_t *y;
    float *h;                                  // [T, R]
    int splits;
};

// Some rows of a sequence and their adapter (-1: none)
struct Tile {
    int row0, rows, a;
};
__device__ __forceinline__ bool rows_of(const AdapterArgs &g, int b, int *s0, int *n)
{
    const int s1 = g.pb.starts[b + 1];
    *s0 = g.pb.starts[b];
    *n = (int)((unsigned)s1 - (unsigned)*s0);
    return *s0 >= 0 && s1 >= *s0 && s1 <= g.pb.T && *n <= g.max_new;
}
__device__ __forceinline__ int adapter_of(const AdapterArgs &g, int b)
{
    const int a = g.ids[b];
    return a >= 0 && a < g.n ? a : -1;
}
__device__ __forceinline__ Tile find_tile(const AdapterArgs &g, int64_t u, int per)
{
    int i, s0, n;
    const int b = g.units.find(g.pb, u, &i);
    if (b >= g.pb.B || !rows_of(g, b, &s0, &n) || (int64_t)i * per >= n) return {0, 0, -1};
    return {s0 + i * per, min(per, n - i * per), adapter_of(g, b)};
}
// names what does not fit together: a workgroup of its own, since such a sequence may have no tile
__device__ void look_over(const AdapterArgs &g)
{
    for (int b = threadIdx.x; b < g.pb.B; b += blockDim.x) {
        int s0, n;
        if (!rows_of(g, b, &s0, &n) || g.ids[b] < -1 || g.ids[b] >= g.n) report(g.pb, b);
    }
}

__device__ __forceinline__ half8_t zero8() { return half8_t{0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ float4_t zero4() { return float4_t{0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ half8_t load8(const half_t *p) { return *reinterpret_cast<const half8_t *>(p); }
__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Exponent of the largest of finite values, whose bits are given, and a power of two
__device__ __forceinline__ int exponent(int bits) { return min(max((bits >> 23) - 127, -126), 126); }
__device__ __forceinline__ float two_to(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }
__device__ __forceinline__ int finite_bits(float v)
{
    const float a = fabsf(v);
    return a < INFINITY ? __builtin_bit_cast(int, a) : 0;
}

// the two f16 terms of a value
__device__ __forceinline__ void two_terms(float v, half_t *hi, half_t *lo)
{
    const half_t a = f2h(v);
    *hi = a;
    *lo = fabsf(h2f(a)) < INFINITY ? f2h(v - h2f(a)) : (half_t)0.f;
}

typedef __fp16 fp16x4_t __attribute__((__vector_size__(4 * sizeof(__fp16))));
// 4 consecutive k of a lane's column out of a [k][column] tile: of the 16 lanes of a group lane l names the 4 columns of piece l & 3
// in row l >> 2, and gets column l
__device__ __forceinline__ half4_t read_tr(const half_t *q)
{
    typedef __attribute__((address_space(3))) fp16x4_t *lds_ptr;
    return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_ptr)q));
}
__device__ __forceinline__ half8_t both(half4_t a, half4_t b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// ---------------------------------------------------------------- h of a tile of 16 rows
// acc[i][e]: row of the tile lane & 15, column 16 i + 4 (lane >> 4) + e of h, over the steps of 32 of the contraction that the wave has.
// W: [R, K] (TR = false) or [K, R] (true), lds: 32 rows of 2 R + 16 bytes of its own for each wave.
template <int RT, int WAVES, bool TR>
__device__ __forceinline__ void tile_h(const half_t *x, int64_t ldx, int rows, int K, const half_t *W, int R, half_t *lds, float4_t (&acc)[RT])
{
    constexpr int U = TR ? (RT <= 2 ? 2 : 1) : RT <= 2 ? 4 : RT <= 4 ? 2 : 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const half_t *xr = x + (int64_t)min(m, rows - 1) * ldx + 8 * g;
    const int pitch = R + 8;
#pragma unroll
    for (int i = 0; i < RT; i++) acc[i] = zero4();
    const int steps = (K + 31) / 32;
    for (int c0 = wave * U; c0 < steps; c0 += WAVES * U) {
        half8_t xf[U], wf[U][RT];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k0 = 32 * (c0 + u);
            xf[u] = load8(xr + min(k0, K - 8 - 8 * g));
            if constexpr (!TR) {
#pragma unroll
                for (int i = 0; i < RT; i++) wf[u][i] = load8(W + (int64_t)min(16 * i + m, R - 1) * K + min(k0 + 8 * g, K - 8));
            } else {
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const int piece = 64 * i + lane, per = R / 8, k = piece / per;
                    wf[u][i] = load8(W + (int64_t)min(k0 + min(k, 31), K - 1) * R + 8 * (piece % per));
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k0 = 32 * (c0 + u);
            if (k0 >= K) break;
            if constexpr (TR) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const int piece = 64 * i + lane, per = R / 8, k = piece / per;
                    if (k < 32) *reinterpret_cast<half8_t *>(lds + k * pitch + 8 * (piece % per)) = k0 + k < K ? wf[u][i] : zero8();
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    // (columns from R on are those of a row of h that is not used; the last piece stays within the row's padding)
                    const half_t *q = lds + (8 * g + (m >> 2)) * pitch + min(16 * i + 4 * (m & 3), R + 4);
                    wf[u][i] = both(read_tr(q), read_tr(q + 4 * pitch));
                }
            }
            if (k0 + 8 * g >= K) {
                xf[u] = zero8();
#pragma unroll
                for (int i = 0; i < RT; i++) wf[u][i] = zero8();
            }
#pragma unroll
            for (int i = 0; i < RT; i++) acc[i] = mfma(wf[u][i], xf[u], acc[i]);
        }
    }
}

// what the waves have of it added up: put(item, row, column, sum) for a thread's items of [16][16 RT]
template <int RT, int WAVES, class Put>
__device__ __forceinline__ void join_h(float *red, const float4_t (&acc)[RT], Put put)
{
    constexpr int C = 16 * RT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < RT; i++)
        *reinterpret_cast<float4_t *>(red + (wave * kTile + (lane & 15)) * C + 16 * i + 4 * (lane >> 4)) = acc[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (kTile * C + 64 * WAVES - 1) / (64 * WAVES); i++) {
        const int e = threadIdx.x + 64 * WAVES * i;
        if (e >= kTile * C) break;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) s += red[w * kTile * C + e];
        put(i, e / C, e % C, s);
    }
}

// ---------------------------------------------------------------- forward
// A workgroup to 16 rows of a sequence and 1 / splits of the columns of y; h is formed by each of them.
template <int RT>
__global__ void __launch_bounds__(512) adapter_kernel(AdapterArgs g)
{
    constexpr int W = 8, C = 16 * RT, HP = 32 * RT + 8;
    __shared__ __attribute__((aligned(16))) float red[W * kTile * C];
    __shared__ __attribute__((aligned(16))) half_t hs[kTile * HP];
    __shared__ int largest[kTile];
    const int64_t blocks = g.units.count * g.splits;
    if (blockIdx.x >= blocks) return look_over(g);
    // the splits of a tile 8 apart, on one XCD: they read the same x and A
    const int64_t group = blockIdx.x / (8 * g.splits), left = min((int64_t)8, g.units.count - 8 * group);
    const int in = (int)(blockIdx.x - 8 * group * g.splits), split = in / (int)left;
    const Tile t = find_tile(g, 8 * group + in % left, kTile);
    if (t.rows == 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q4 = lane >> 4;
    const int R = g.R, K = g.K, N = g.N;
    const float scale = t.a < 0 ? 0.f : g.scale[t.a];
    if (t.a < 0) {                             // no adapter
        if (split == 0)
            for (int e = threadIdx.x; e < t.rows * R; e += 64 * W) g.h[(int64_t)t.row0 * R + e] = 0.f;
        if (g.base == g.y) return;
        for (int e = split * 64 * W + threadIdx.x; e < t.rows * (N / 8); e += g.splits * 64 * W) {
            const int64_t r = t.row0 + e / (N / 8);
            const int c = 8 * (e % (N / 8));
            *reinterpret_cast<half8_t *>(g.y + r * g.ldy + c) = g.base ? load8(g.base + r * g.ldb + c) : zero8();
        }
        return;
    }
    float4_t acc[RT];
    tile_h<RT, W, false>(g.x + t.row0 * g.ldx, g.ldx, t.rows, K, g.A + (int64_t)t.a * R * K, R, nullptr, acc);
    for (int e = threadIdx.x; e < kTile * HP / 8; e += 64 * W) *reinterpret_cast<half8_t *>(hs + 8 * e) = zero8();
    if (threadIdx.x < kTile) largest[threadIdx.x] = 0;
    float sum[(RT + 1) / 2];
    join_h<RT, W>(red, acc, [&](int i, int r, int c, float s) __attribute__((always_inline)) {
        sum[i] = s;
        if (c >= R) return;
        atomicMax(largest + r, finite_bits(s));
        if (split == 0 && r < t.rows) g.h[(int64_t)(t.row0 + r) * R + c] = s;
    });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (RT + 1) / 2; i++) {
        const int e = threadIdx.x + 64 * W * i, r = e / C, c = e % C;
        if (e < kTile * C && c < R) two_terms(sum[i] * two_to(-exponent(largest[r])), hs + r * HP + c, hs + r * HP + R + c);
    }
    __syncthreads();
    const float up = two_to(exponent(largest[m]));
    half8_t hf[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) hf[i] = load8(hs + m * HP + 32 * i + 8 * q4);
    // a wave to 64 columns: rows of B in an order that leaves a lane 16 columns of its row side by side
    const half_t *B = g.B + (int64_t)t.a * N * R;
    for (int n0 = 64 * (split * W + wave); n0 < N; n0 += 64 * W * g.splits) {
        float4_t o[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            o[j] = zero4();
            const half_t *row = B + (int64_t)min(n0 + 16 * (m >> 2) + 4 * j + (m & 3), N - 1) * R;
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const int kk = 32 * i + 8 * q4;
                half8_t w = load8(row + (kk < R ? kk : kk < 2 * R ? kk - R : 0));
                w = kk < 2 * R ? w : zero8();
                o[j] = mfma(w, hf[i], o[j]);
            }
        }
        if (m >= t.rows) continue;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const int c = n0 + 16 * q4 + 8 * p;
            if (c >= N) break;
            half8_t v;
            if (g.base) {
                v = load8(g.base + (t.row0 + m) * g.ldb + c);
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = f2h(h2f(v[k]) + scale * (up * o[2 * p + k / 4][k % 4]));
            } else
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = f2h(scale * (up * o[2 * p + k / 4][k % 4]));
            *reinterpret_cast<half8_t *>(g.y + (t.row0 + m) * g.ldy + c) = v;
        }
    }
}

// ---------------------------------------------------------------- gradients
constexpr int kRows = 64, kCols = 128;         // rows and columns of a step of the second kernel

struct GradArgs {
    AdapterArgs f;                             // x, A, B, h as in the forward pass; y, ldy: dx; base: what it is added to, or null
    const half_t *dy;
    int64_t lddy;
    float *dh;                                 // [T, R], without the scale
    int *rows, *begin;                         // rows of adapter a: rows[begin[a]] .. rows[begin[a + 1] - 1]
    float *parts;                              // of dA [R, K] and dB [N, R], a block of rows each
    half_t *dA, *dB;
    int dA_acc, dB_acc, per;                   // rows of a block
    int64_t blocks;
};

// The rows of each adapter, sequence after sequence, by one workgroup of 8 waves.  A wave to an adapter.  (Sums no larger than T:
// sequences that overlap may have more rows than there are.)
constexpr int kMaxAdapters = 1024;
__device__ void plan(const GradArgs &d, int *counts)
{
    const AdapterArgs &g = d.f;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int a = wave; a < g.n; a += 8) {
        int c = 0;
        for (int b0 = 0; b0 < g.pb.B; b0 += 64) {
            int s0, n;
            const int b = min(b0 + lane, g.pb.B - 1);
            if (b0 + lane < g.pb.B && rows_of(g, b, &s0, &n) && adapter_of(g, b) == a) c = min(c + n, g.pb.T);
        }
        for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o);
        if (lane == 0) counts[a] = min(c, g.pb.T);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int s = 0;
        for (int a = 0; a < g.n; a++) {
            const int c = counts[a];
            counts[a] = s;
            s = min(s + c, g.pb.T);
        }
        counts[g.n] = s;
    }
    __syncthreads();
    for (int a = threadIdx.x; a <= g.n; a += 512) d.begin[a] = counts[a];
    for (int a = wave; a < g.n; a += 8) {
        int at = counts[a];
        for (int b0 = 0; b0 < g.pb.B; b0 += 64) {
            int s0 = 0, n = 0;
            const int b = min(b0 + lane, g.pb.B - 1);
            const bool mine = b0 + lane < g.pb.B && rows_of(g, b, &s0, &n) && adapter_of(g, b) == a;
            uint64_t todo = __ballot(mine && n > 0);
            while (todo) {
                const int l = __builtin_ctzll(todo);
                todo &= todo - 1;
                const int first = __builtin_amdgcn_readlane(s0, l), count = __builtin_amdgcn_readlane(n, l);
                for (int i = lane; i < count && at + i < g.pb.T; i += 64) d.rows[at + i] = first + i;
                at = min(at + count, g.pb.T);
            }
        }
    }
}

// dh of 16 rows of a sequence; dx of rows without an adapter.  The last two workgroups: the plan, and what does not fit.
template <int RT>
__global__ void __launch_bounds__(512) dh_kernel(GradArgs d)
{
    constexpr int W = 8, C = 16 * RT;
    __shared__ __attribute__((aligned(16))) float red[W * kTile * C];
    __shared__ __attribute__((aligned(16))) half_t lds[W][32 * (C + 8)];
    __shared__ int counts[kMaxAdapters + 1];
    const AdapterArgs &g = d.f;
    if (blockIdx.x == 0) return plan(d, counts);
    const int64_t u = (int64_t)blockIdx.x - 1;
    if (u >= g.units.count) return look_over(g);
    const Tile t = find_tile(g, u, kTile);
    if (t.rows == 0) return;
    const int R = g.R, K = g.K;
    if (t.a < 0) {
        if (g.base) return;                    // (added to: nothing)
        for (int e = threadIdx.x; e < t.rows * (K / 8); e += 64 * W)
            *reinterpret_cast<half8_t *>(g.y + (int64_t)(t.row0 + e / (K / 8)) * g.ldy + 8 * (e % (K / 8))) = zero8();
        return;
    }
    float4_t acc[RT];
    tile_h<RT, W, true>(d.dy + t.row0 * d.lddy, d.lddy, t.rows, g.N, g.B + (int64_t)t.a * g.N * R, R, lds[threadIdx.x >> 6], acc);
    join_h<RT, W>(red, acc, [&](int, int r, int c, float s) __attribute__((always_inline)) {
        if (c < R && r < t.rows) d.dh[(int64_t)(t.row0 + r) * R + c] = s;
    });
}

// units of adapter a begin at begin[a] / per + a
__device__ __forceinline__ int64_t unit_of(const GradArgs &d, int a) { return (int64_t)(d.begin[a] / d.per) + a; }

// A block of an adapter's rows and 128 columns: of x, for dx and the block's part of dA, or of dy, for its part of dB.
template <int RT>
__global__ void __launch_bounds__(256) grad_kernel(GradArgs d)
{
    constexpr int HP = 32 * RT + 8, XP = kCols + 16;
    __shared__ __attribute__((aligned(16))) half_t xs[kRows * XP], hs[kRows * HP], hr[kRows * HP], as[16 * RT * XP];
    __shared__ int largest[2][kRows];
    const AdapterArgs &g = d.f;
    const int R = g.R, K = g.K, N = g.N, kchunks = (K + kCols - 1) / kCols, chunks = kchunks + (N + kCols - 1) / kCols;
    const int64_t u = blockIdx.x / chunks;
    const int chunk = (int)(blockIdx.x % chunks);
    const bool of_x = chunk < kchunks;
    const int c0 = kCols * (of_x ? chunk : chunk - kchunks), width = of_x ? K : N;
    // (unit 0 is adapter 0's: one more than the adapters that begin behind it)
    const int a = count_below(g.n - 1, u, [&](int i) { return unit_of(d, i); });
    const int first = d.begin[a] + (int)(u - unit_of(d, a)) * d.per, count = min(d.per, d.begin[a + 1] - first);
    if (count <= 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q4 = lane >> 4;
    const float scale = g.scale[a];
    const half_t *src = of_x ? g.x : d.dy;
    const int64_t ld = of_x ? g.ldx : d.lddy;
    const float *hsrc = of_x ? d.dh : g.h;
    if (of_x)
        for (int e = threadIdx.x; e < 16 * RT * (kCols / 8); e += 256) {
            const int r = e / (kCols / 8), c = 8 * (e % (kCols / 8));
            *reinterpret_cast<half8_t *>(as + r * XP + c) = r < R && c0 + c < K ? load8(g.A + ((int64_t)a * R + r) * K + c0 + c) : zero8();
        }
    for (int e = threadIdx.x; e < kRows * HP / 8; e += 256)
        *reinterpret_cast<half8_t *>(hs + 8 * e) = *reinterpret_cast<half8_t *>(hr + 8 * e) = zero8();
    if (threadIdx.x < kRows) largest[0][threadIdx.x] = 0;
    float4_t acc[RT][2];
#pragma unroll
    for (int i = 0; i < RT; i++) acc[i][0] = acc[i][1] = zero4();
    int top = -126;                            // exponent that the sums are scaled by
    for (int r0 = 0, turn = 0; r0 < count; r0 += kRows, turn ^= 1) {
        __syncthreads();
        if (threadIdx.x < kRows) largest[turn ^ 1][threadIdx.x] = 0;
        for (int e = threadIdx.x; e < kRows * (kCols / 8); e += 256) {
            const int r = e / (kCols / 8), c = 8 * (e % (kCols / 8));
            *reinterpret_cast<half8_t *>(xs + r * XP + c) =
                r0 + r < count && c0 + c < width ? load8(src + (int64_t)d.rows[first + r0 + r] * ld + c0 + c) : zero8();
        }
        float4_t v[RT];
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int e = threadIdx.x + 256 * i, r = e / (R / 4), c = 4 * (e % (R / 4));
            if (r >= kRows) break;
            v[i] = r0 + r < count ? *reinterpret_cast<const float4_t *>(hsrc + (int64_t)d.rows[first + r0 + r] * R + c) : zero4();
            atomicMax(&largest[turn][r], max(max(finite_bits(v[i][0]), finite_bits(v[i][1])), max(finite_bits(v[i][2]), finite_bits(v[i][3]))));
        }
        __syncthreads();
        const int now = max(top, exponent(__builtin_bit_cast(int, wave_max(__builtin_bit_cast(float, largest[turn][lane])))));
        const float less = two_to(max(top - now, -126));
        top = now;
#pragma unroll
        for (int i = 0; i < RT; i++) acc[i][0] *= less, acc[i][1] *= less;
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int e = threadIdx.x + 256 * i, r = e / (R / 4), c = 4 * (e % (R / 4));
            if (r >= kRows) break;
            const float all = two_to(-top), own = two_to(-exponent(largest[turn][r]));
#pragma unroll
            for (int k = 0; k < 4; k++) {
                two_terms(v[i][k] * all, hs + r * HP + c + k, hs + r * HP + R + c + k);
                if (of_x) two_terms(v[i][k] * own, hr + r * HP + c + k, hr + r * HP + R + c + k);
            }
        }
        __syncthreads();
        // the sums over rows: step s has rows 32 s + 4 q4 + 0 .. 3 and those 16 further, in both operands
#pragma unroll
        for (int s = 0; s < kRows / 32; s++) {
            const int row = 32 * s + 4 * q4 + (m >> 2);
            half8_t xf[2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const half_t *q = xs + row * XP + 32 * wave + 16 * c + 4 * (m & 3);
                xf[c] = both(read_tr(q), read_tr(q + 16 * XP));
            }
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const half_t *q = hs + row * HP + p * R + 16 * i + 4 * (m & 3);
                    const half8_t hf = both(read_tr(q), read_tr(q + 16 * HP));
#pragma unroll
                    for (int c = 0; c < 2; c++) acc[i][c] = of_x ? mfma(hf, xf[c], acc[i][c]) : mfma(xf[c], hf, acc[i][c]);
                }
        }
        if (!of_x) continue;
        // dx of 32 columns a wave, 8 of them side by side in a lane
#pragma unroll
        for (int t = 0; t < kRows / 16; t++) {
            float4_t o[2] = {zero4(), zero4()};
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const int kk = 32 * i + 8 * q4, r = kk < R ? kk : kk < 2 * R ? kk - R : 0;
                const half8_t hf = load8(hr + (16 * t + m) * HP + kk);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const half_t *q = as + (r + (m >> 2)) * XP + 32 * wave + 8 * (m & 3) + 4 * j;
                    half8_t w = both(read_tr(q), read_tr(q + 4 * XP));
                    w = kk < 2 * R ? w : zero8();
                    o[j] = mfma(w, hf, o[j]);
                }
            }
            const int r = r0 + 16 * t + m, c = c0 + 32 * wave + 8 * q4;
            if (r >= count || c >= K) continue;
            const int64_t row = d.rows[first + r];
            const float up = two_to(exponent(largest[turn][16 * t + m]));
            half8_t v;
            if (g.base) {
                v = load8(g.base + row * g.ldb + c);
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = f2h(h2f(v[k]) + scale * (up * o[k / 4][k % 4]));
            } else
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = f2h(scale * (up * o[k / 4][k % 4]));
            *reinterpret_cast<half8_t *>(g.y + row * g.ldy + c) = v;
        }
    }
    const float up = two_to(top);
    float *part = d.parts + u * R * (K + N);
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (of_x) {
                    const int r = 16 * i + 4 * q4 + e, k = c0 + 32 * wave + 16 * c + m;
                    if (r < R && k < K) part[(int64_t)r * K + k] = up * acc[i][c][e];
                } else {
                    const int n = c0 + 32 * wave + 16 * c + 4 * q4 + e, r = 16 * i + m;
                    if (r < R && n < N) part[(int64_t)R * K + (int64_t)n * R + r] = up * acc[i][c][e];
                }
            }
}

// The blocks' parts of an adapter's gradients added up, 4 elements to a thread
__global__ void __launch_bounds__(256) join_kernel(GradArgs d)
{
    const AdapterArgs &g = d.f;
    const int a = blockIdx.y;
    const int64_t size = (int64_t)g.R * (g.K + g.N), e = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x), ofA = (int64_t)g.R * g.K;
    if (e >= size) return;
    const bool isA = e < ofA;
    half_t *to = isA ? d.dA + a * ofA + e : d.dB + (int64_t)a * g.R * g.N + (e - ofA);
    const bool acc = isA ? d.dA_acc : d.dB_acc;
    const int count = d.begin[a + 1] - d.begin[a], parts = (count + d.per - 1) / d.per;
    if (parts == 0 && acc) return;
    const float *p = d.parts + unit_of(d, a) * size + e;
    float4_t s = zero4();
    for (int i = 0; i < parts; i++) s += *reinterpret_cast<const float4_t *>(p + i * size);
    const float scale = g.scale[a];
    half4_t v = acc ? *reinterpret_cast<const half4_t *>(to) : half4_t{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = parts == 0 ? (half_t)0.f : acc ? f2h(h2f(v[k]) + scale * s[k]) : f2h(scale * s[k]);
    *reinterpret_cast<half4_t *>(to) = v;
}

// ---------------------------------------------------------------- host
int check(const char *who, int64_t T, int64_t S, int64_t K, int64_t N, int64_t R, int64_t n, int64_t max_new, const void *x, int64_t ldx,
          const void *A, const void *B, const void *starts, const void *ids, const void *scale, const void *status, AdapterArgs *g)
{
    CACTI_REQUIRE(T > 0 && S > 0 && K > 0 && N > 0 && R > 0 && n > 0 && max_new > 0, CACTI_E_INVALID, "%s: empty shape", who);
    CACTI_REQUIRE(x && A && B && starts && ids && scale, CACTI_E_INVALID, "%s: null pointer", who);
    CACTI_REQUIRE(R % 8 == 0 && R <= kMaxR, CACTI_E_NOTIMPL, "%s: need R %% 8 == 0 and R <= %d", who, kMaxR);
    CACTI_REQUIRE(K % 8 == 0 && N % 8 == 0 && K <= (1 << 20) && N <= (1 << 20), CACTI_E_NOTIMPL, "%s: need K and N multiples of 8, at most 2^20", who);
    CACTI_REQUIRE(T <= (1 << 24) && S <= (1 << 20) && n <= kMaxAdapters, CACTI_E_NOTIMPL, "%s: at most 2^24 rows, 2^20 sequences, %d adapters", who,
                  kMaxAdapters);
    CACTI_REQUIRE(ldx >= K && ldx % 8 == 0, CACTI_E_INVALID, "%s: row pitch of x below a row, or no multiple of 8", who);
    CACTI_REQUIRE(aligned(x, 16) && aligned(A, 16) && aligned(B, 16) && aligned(starts, 4) && aligned(ids, 4) && aligned(scale, 4) && aligned(status, 4),
                  CACTI_E_INVALID, "%s: operands must be 16-byte aligned", who);
    *g = AdapterArgs{};
    g->pb.T = (int)T;
    g->pb.B = (int)S;
    g->pb.starts = (const int *)starts;
    g->pb.status = (int *)const_cast<void *>(status);
    g->max_new = (int)(max_new < T ? max_new : T);
    g->units = make_units(T, S, kTile, 1, 1, (g->max_new + kTile - 1) / kTile);
    g->K = (int)K, g->N = (int)N, g->R = (int)R, g->n = (int)n;
    g->x = (const half_t *)x, g->A = (const half_t *)A, g->B = (const half_t *)B;
    g->ids = (const int *)ids, g->scale = (const float *)scale;
    g->ldx = ldx;
    return 0;
}

// RT of 1, 2, 4 or 8: R rounded up to 16 of them
#define CACTI_BY_RANK(R, launch)        \
    do {                                \
        if ((R) <= 16) launch(1);       \
        else if ((R) <= 32) launch(2);  \
        else if ((R) <= 64) launch(4);  \
        else launch(8);                 \
    } while (0)

// rows of a block: some hundred workgroups at least, and no more parts than that needs
int64_t block_rows(int64_t T, int64_t K, int64_t N)
{
    const int64_t chunks = (K + kCols - 1) / kCols + (N + kCols - 1) / kCols, steps = (T + kRows - 1) / kRows;
    int64_t per = steps * chunks / 768;
    per = per < 1 ? 1 : per > 64 ? 64 : per;
    return per * kRows;
}

struct Workspace {
    size_t dh, rows, begin, parts, bytes;
    int64_t per, blocks;
};
Workspace workspace(int64_t T, int64_t K, int64_t N, int64_t R, int64_t n)
{
    Workspace w;
    auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    w.per = block_rows(T, K, N);
    w.blocks = T / w.per + n;
    w.dh = 0;
    w.rows = w.dh + up((size_t)T * R * 4);
    w.begin = w.rows + up((size_t)T * 4);
    w.parts = w.begin + up((size_t)(n + 1) * 4);
    w.bytes = w.parts + (size_t)w.blocks * R * (K + N) * 4;
    return w;
}

}  // namespace

CACTI_API int cacti_hip_adapter_fwd(int64_t T, int64_t S, int64_t K, int64_t N, int64_t R, int64_t n, int64_t max_new, const void *x, int64_t ldx,
                                    const void *A, const void *B, const void *starts, const void *ids, const void *scale, const void *base,
                                    int64_t ldb, void *y, int64_t ldy, void *h, void *status, void *stream)
{
    AdapterArgs g;
    const int rc = check("adapter_fwd", T, S, K, N, R, n, max_new, x, ldx, A, B, starts, ids, scale, status, &g);
    if (rc) return rc;
    CACTI_REQUIRE(y && h, CACTI_E_INVALID, "adapter_fwd: null pointer");
    CACTI_REQUIRE(aligned(y, 16) && aligned(base, 16) && aligned(h, 16), CACTI_E_INVALID, "adapter_fwd: operands must be 16-byte aligned");
    CACTI_REQUIRE(ldy >= N && ldy % 8 == 0 && (!base || (ldb >= N && ldb % 8 == 0)), CACTI_E_INVALID,
                  "adapter_fwd: row pitch below a row, or no multiple of 8");
    CACTI_REQUIRE(!rows_share(T, x, ldx, K, y, ldy, N), CACTI_E_INVALID, "adapter_fwd: y shares memory with x");
    CACTI_REQUIRE(!base || (base == y && ldb == ldy) || !rows_share(T, base, ldb, N, y, ldy, N), CACTI_E_INVALID,
                  "adapter_fwd: y takes the base's place, with the same pitch, or shares no memory with it");
    g.base = (const half_t *)base, g.ldb = ldb;
    g.y = (half_t *)y, g.ldy = ldy;
    g.h = (float *)h;
    // (columns are split until the device is full: 512 of them are an iteration of a workgroup)
    const int64_t most = (N + 511) / 512, want = (device_cus() + g.units.count - 1) / g.units.count;
    g.splits = (int)(want < 1 ? 1 : want < most ? want : most);
    const int64_t blocks = g.units.count * g.splits + (status ? 1 : 0);
    CACTI_REQUIRE(blocks <= INT32_MAX, CACTI_E_NOTIMPL, "adapter_fwd: too many tiles");
#define LAUNCH(RT) hipLaunchKernelGGL((adapter_kernel<RT>), dim3((unsigned)blocks), dim3(512), 0, (hipStream_t)stream, g)
    CACTI_BY_RANK(R, LAUNCH);
#undef LAUNCH
    return launch_status("adapter_fwd");
}

CACTI_API size_t cacti_hip_adapter_bwd_workspace(int64_t T, int64_t K, int64_t N, int64_t R, int64_t n)
{
    return T > 0 && K > 0 && N > 0 && R > 0 && n > 0 ? workspace(T, K, N, R, n).bytes : 0;
}

CACTI_API int cacti_hip_adapter_bwd(int64_t T, int64_t S, int64_t K, int64_t N, int64_t R, int64_t n, int64_t max_new, const void *x, int64_t ldx,
                                    const void *A, const void *B, const void *starts, const void *ids, const void *scale, const void *h,
                                    const void *dy, int64_t lddy, void *dx, int64_t lddx, int dx_acc, void *dA, int dA_acc, void *dB, int dB_acc,
                                    void *ws, size_t ws_bytes, void *status, void *stream)
{
    GradArgs d{};
    const int rc = check("adapter_bwd", T, S, K, N, R, n, max_new, x, ldx, A, B, starts, ids, scale, status, &d.f);
    if (rc) return rc;
    CACTI_REQUIRE(h && dy && dx && dA && dB && ws, CACTI_E_INVALID, "adapter_bwd: null pointer");
    CACTI_REQUIRE(aligned(h, 16) && aligned(dy, 16) && aligned(dx, 16) && aligned(dA, 16) && aligned(dB, 16) && aligned(ws, 16), CACTI_E_INVALID,
                  "adapter_bwd: operands must be 16-byte aligned");
    CACTI_REQUIRE(lddy >= N && lddy % 8 == 0 && lddx >= K && lddx % 8 == 0, CACTI_E_INVALID, "adapter_bwd: row pitch below a row, or no multiple of 8");
    CACTI_REQUIRE(!rows_share(T, x, ldx, K, dx, lddx, K) && !rows_share(T, dy, lddy, N, dx, lddx, K), CACTI_E_INVALID,
                  "adapter_bwd: dx shares memory with x or dy");
    const Workspace w = workspace(T, K, N, R, n);
    CACTI_REQUIRE(ws_bytes >= w.bytes, CACTI_E_INVALID, "adapter_bwd: workspace of %zu bytes, %zu needed", ws_bytes, w.bytes);
    const int64_t chunks = (K + kCols - 1) / kCols + (N + kCols - 1) / kCols, size = R * (K + N);
    CACTI_REQUIRE(w.blocks * chunks <= INT32_MAX, CACTI_E_NOTIMPL, "adapter_bwd: too many tiles");
    char *p = (char *)ws;
    d.f.h = (float *)const_cast<void *>(h);
    d.f.y = (half_t *)dx, d.f.ldy = lddx;
    d.f.base = dx_acc ? (const half_t *)dx : nullptr, d.f.ldb = lddx;
    d.dy = (const half_t *)dy, d.lddy = lddy;
    d.dh = (float *)(p + w.dh);
    d.rows = (int *)(p + w.rows), d.begin = (int *)(p + w.begin);
    d.parts = (float *)(p + w.parts);
    d.dA = (half_t *)dA, d.dB = (half_t *)dB, d.dA_acc = dA_acc, d.dB_acc = dB_acc;
    d.per = (int)w.per, d.blocks = w.blocks;
    const unsigned tiles = (unsigned)(d.f.units.count + 1 + (status ? 1 : 0));
#define LAUNCH(RT)                                                                                                                   \
    do {                                                                                                                             \
        hipLaunchKernelGGL((dh_kernel<RT>), dim3(tiles), dim3(512), 0, (hipStream_t)stream, d);                                      \
        hipLaunchKernelGGL((grad_kernel<RT>), dim3((unsigned)(w.blocks * chunks)), dim3(256), 0, (hipStream_t)stream, d);            \
    } while (0)
    CACTI_BY_RANK(R, LAUNCH);
#undef LAUNCH
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)((size + 1023) / 1024), (unsigned)n), dim3(256), 0, (hipStream_t)stream, d);
    return launch_status("adapter_bwd");
}
