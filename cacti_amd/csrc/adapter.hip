// Low-rank adapters of many requests beside a shared projection, and their gradients.  Row t of sequence s, with the adapter
// a = ids[s] (A_a [R, K], B_a [N, R], scale_a):
//   h = A_a x,  y = base + scale_a B_a h
//   dh = B_a^T dy,  dx = scale_a A_a^T dh,  dA_a = scale_a sum_t dh x^T,  dB_a = scale_a sum_t dy h^T   (over a's rows)
//
// All sums are fp32 (matrix instructions).  h and dh are one operand of a second product: they meet it as two f16 terms, value
// and what its rounding left, 22 bits in all, so that results are rounded once.  They are scaled by a power of two first, that of the
// largest of a row (for y and dx) or of the rows so far (for dA and dB): a gradient may lie far below f16's range and h beyond it.
// The terms lie side by side as 2 R columns, which for R = 16 fill the 32 that an instruction takes.
//
// A matrix instruction wants 16 rows in 16 lanes side by side.  Loads in that order take 64 looks at the cache each, a quarter of what a
// compute unit can read (measured: 26 GB/s of it); here 4 lanes read 64 bytes of a row, and a wave turns its tiles of 16 rows of 64
// bytes in LDS, on the way in and on the way out.
//
// What bounds it, with times on the device, 3200 to 3200, R = 16 where nothing else is said.  A few rows: the chain of a launch, numbers of
// the sequence, x and A, the sum over the waves, B (one row 6.5 us, 64 sequences of up to 5 rows 8.1).  Many: memory.  2227 rows, 3200 to
// 8640, R = 64: h 10.1 us, y 22.1 for 77 MB of base and y, 3.5 TB/s; between loads and stores stand the turns in LDS.  The adjoint of 4096
// rows: 9.8 us for the terms of dh and h (dy read once), 18.0 for dx and the parts of dA and dB (79 MB, 4.4 TB/s), 3.9 to join those;
// 269 rows of 1024 to 2816 take 7.7, 5.9 and 3.8, little more than launches.  R = 128: 24, 44 and 7, of those 44 the matrix pipe 8, vector
// operations 12 and LDS 13 (every wave reads and scales all terms for its 32 columns), which two waves to a SIMD do not bring together; the 24
// are those of B, read and turned for every 16 rows.
#include <algorithm>
#include <initializer_list>

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
__device__ __forceinline__ Tile find_tile(const AdapterArgs &g, int u, int per)
{
    int i, s0, n, b;
    if (g.units.even) b = u / g.units.even, i = u - b * g.units.even;
    else b = g.units.find(g.pb, u, &i);
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

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ __forceinline__ half8_t zero8() { return half8_t{0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ float4_t zero4() { return float4_t{0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ half8_t load8(const half_t *p) { return *reinterpret_cast<const half8_t *>(p); }
__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Values are scaled so that the largest is in 2^kTop .. 2^(kTop + 1): exponent that the largest of finite values, whose bits are given, has
// beyond that; a power of two
constexpr int kTop = 10;
__device__ __forceinline__ int exponent(int bits) { return min(max((bits >> 23) - 127, -100), 126) - kTop; }
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

// ---------------------------------------------------------------- tiles of 16 rows of 64 bytes, a wave's own
// A lane's 16 bytes of one, row lane / 4 as it lies in memory or row lane % 16 as an operand; where in LDS they are, without conflicts
// in either order.
constexpr int kTileHalves = 16 * 32;
__device__ __forceinline__ int mem_row() { return (threadIdx.x & 63) >> 2; }
__device__ __forceinline__ int mem_col() { return 8 * (threadIdx.x & 3); }
__device__ __forceinline__ int place(int row, int piece) { return 32 * row + 8 * (piece ^ (row >> 2)); }
__device__ __forceinline__ half_t *as_memory(half_t *tile) { return tile + place(mem_row(), threadIdx.x & 3); }
__device__ __forceinline__ half_t *as_operand(half_t *tile)
{
    const int lane = threadIdx.x & 63;
    return tile + place(lane & 15, lane >> 4);
}
__device__ __forceinline__ void put8(half_t *p, half8_t v) { *reinterpret_cast<half8_t *>(p) = v; }
// Waits for what a register is loaded with.  (Where a path goes by without a use of it the compiler waits before the register's next load, and for
// all stores under way with it.)
__device__ __forceinline__ void arrived(half8_t &v) { asm volatile("" : "+v"(v)); }
// what a wave's lanes have written to LDS before is there for its lanes after (they take turns in order)
__device__ __forceinline__ void in_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// ---------------------------------------------------------------- h of a tile of 16 TB rows
// acc[t][i][e]: row 16 t + (lane & 15) of the tile, column 16 i + 4 (lane >> 4) + e of h, over those of steps s0 .. s1 - 1 of 32 that the wave
// has.  W: [R, K] (TR = false) or [K, R] (true); lds: kLds halves, the wave's own.  Loads are a turn ahead.
template <int RT, int TB, int WAVES, bool TR>
struct TileH {
    static constexpr int U = RT + TB <= 2 && WAVES <= 8 ? 4 : RT + TB <= 6 ? 2 : 1, kLds = TB * kTileHalves + (TR ? 32 * (16 * RT + 8) : RT * kTileHalves);
    const half_t *xr[TB], *W;
    int K, R, m, g;
    half_t *lds;
    float4_t acc[TB][RT];
    struct Turn {
        half8_t x[U][TB], w[U][RT];
    };
    __device__ __forceinline__ TileH(const half_t *x, int64_t ldx, int rows, int k, const half_t *w, int r, half_t *l) : W(w), K(k), R(r), lds(l)
    {
        const int lane = threadIdx.x & 63;
        m = lane & 15, g = lane >> 4;
#pragma unroll
        for (int t = 0; t < TB; t++) {
            xr[t] = x + (int64_t)min(16 * t + mem_row(), rows - 1) * ldx;
#pragma unroll
            for (int i = 0; i < RT; i++) acc[t][i] = zero4();
        }
    }
    // (a load behind a branch would be one that is waited for with all later ones: what there is not is some other step)
    __device__ __forceinline__ void load(Turn &o, int c0) const
    {
        const int lane = threadIdx.x & 63;
        // (both halves of a cache line one after the other)
#pragma unroll
        for (int t = 0; t < TB; t++)
#pragma unroll
            for (int u = 0; u < U; u++) o.x[u][t] = load8(xr[t] + min(32 * (c0 + u) + mem_col(), K - 8));
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k0 = 32 * (c0 + u);
                if constexpr (!TR) o.w[u][i] = load8(W + (int64_t)min(16 * i + mem_row(), R - 1) * K + min(k0 + mem_col(), K - 8));
                else {
                    const int piece = 64 * i + lane, per = R / 8, k = piece / per;
                    o.w[u][i] = load8(W + (int64_t)min(k0 + min(k, 31), K - 1) * R + 8 * (piece % per));
                }
            }
    }
    __device__ __forceinline__ void add(Turn &o, int c0, int s1)
    {
        const int lane = threadIdx.x & 63, pitch = R + 8;
        half_t *const wl = lds + TB * kTileHalves;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k0 = 32 * (c0 + u);
            if (c0 + u >= s1) break;
            if (k0 + 32 > K && k0 + mem_col() >= K) {
#pragma unroll
                for (int t = 0; t < TB; t++) o.x[u][t] = zero8();
                if constexpr (!TR)
#pragma unroll
                    for (int i = 0; i < RT; i++) o.w[u][i] = zero8();
            }
            in_order();
#pragma unroll
            for (int t = 0; t < TB; t++) put8(as_memory(lds + t * kTileHalves), o.x[u][t]);
#pragma unroll
            for (int i = 0; i < RT; i++) {
                if constexpr (!TR) put8(as_memory(wl + i * kTileHalves), o.w[u][i]);
                else {
                    const int piece = 64 * i + lane, per = R / 8, k = piece / per;
                    if (k < 32) put8(wl + k * pitch + 8 * (piece % per), k0 + k < K ? o.w[u][i] : zero8());
                }
            }
            in_order();
            half8_t xf[TB];
#pragma unroll
            for (int t = 0; t < TB; t++) xf[t] = load8(as_operand(lds + t * kTileHalves));
#pragma unroll
            for (int i = 0; i < RT; i++) {
                half8_t wf;
                if constexpr (!TR) wf = load8(as_operand(wl + i * kTileHalves));
                else {
                    // (columns from R on are those of a row of h that is not used; the last piece stays within the row's padding)
                    const half_t *q = wl + (8 * g + (m >> 2)) * pitch + min(16 * i + 4 * (m & 3), R + 4);
                    wf = both(read_tr(q), read_tr(q + 4 * pitch));
                }
#pragma unroll
                for (int t = 0; t < TB; t++) acc[t][i] = mfma(wf, xf[t], acc[t][i]);
            }
        }
    }
    __device__ __forceinline__ void run(int s0, int s1)
    {
        constexpr int stride = U * WAVES;
        Turn a, b;
        int c = s0 + U * wave_id();
        if (c >= s1) return;
        load(a, c);
        for (; c + 2 * stride < s1; c += 2 * stride) {
            load(b, c + stride);
            add(a, c, s1);
            load(a, c + 2 * stride);
            add(b, c + stride, s1);
        }
        if (c + stride < s1) {
            load(b, c + stride);
            add(a, c, s1);
            add(b, c + stride, s1);
        } else
            add(a, c, s1);
    }
    // what the waves have of it added up: put(item, row, column, sum) for a thread's items of [16 TB][16 RT]
    static constexpr int kItems = (16 * TB * 16 * RT + 64 * WAVES - 1) / (64 * WAVES);
    template <class Put>
    __device__ __forceinline__ void join(float *red, Put put)
    {
        constexpr int C = 16 * RT, all = 16 * TB * C;
        const int wave = threadIdx.x >> 6;
        __syncthreads();                       // (red takes the place of the waves' tiles)
#pragma unroll
        for (int t = 0; t < TB; t++)
#pragma unroll
            for (int i = 0; i < RT; i++) *reinterpret_cast<float4_t *>(red + wave * all + (16 * t + m) * C + 16 * i + 4 * g) = acc[t][i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kItems; i++) {
            const int e = threadIdx.x + 64 * WAVES * i;
            if (e >= all) break;
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) s += red[w * all + e];
            put(i, e / C, e % C, s);
        }
    }
};

// ---------------------------------------------------------------- forward
// h of a row in LDS: its two terms, the second one 16 RT columns behind the first, zeros from R on in either.  RT = 1: both within the 32
// columns of one instruction, which B (or A) meets twice.
template <int RT>
struct Terms {
    static constexpr int kPitch = 32 * RT + 8, kLo = 16 * RT, kN = RT == 1 ? 1 : RT / 2, kM = RT == 1 ? 1 : 2;
    // the row of B that a lane's 8 values of operand i begin at; the columns of h that they meet, part p of kM
    __device__ __forceinline__ static int of(int i, int q4) { return RT == 1 ? 8 * (q4 & 1) : 32 * i + 8 * q4; }
    __device__ __forceinline__ static int column(int i, int p, int q4) { return p * kLo + 32 * i + 8 * q4; }
    __device__ __forceinline__ static void put(half_t *row, int c, float v) { two_terms(v, row + c, row + kLo + c); }
    __device__ __forceinline__ static void clear(half_t *h, int rows)
    {
        for (int e = threadIdx.x; e < rows * kPitch / 8; e += blockDim.x) *reinterpret_cast<half8_t *>(h + 8 * e) = zero8();
    }
};

// Scale of a row's results: the adapter's and what its h was scaled by.  (Within fp32's range, so that it does not make a 0 a NaN: what it is
// multiplied with is 0 or no less than 2^-48, which f16 takes for infinite either way.)
__device__ __forceinline__ float factor_of(float scale, int exp)
{
    const float f = scale * two_to(max(exp, -126));
    return fabsf(f) < INFINITY || fabsf(scale) == INFINITY || scale != scale ? f : copysignf(3.4028234664e38f, f);
}

// Results of a tile of 16 rows and 32 columns to memory, as they are or added to what `old`, as it came from memory, holds: o[j] those of
// row lane & 15, columns 8 (lane >> 4) + 4 j ..; returns the lane's 16 bytes of row mem_row(), columns mem_col() ..  (Turned as fp32 instead,
// in one trip and two tiles at a time: the same for y, and LDS for a workgroup less in the gradients, 22.7 -> 26.8 us.)
template <bool BASE>
__device__ __forceinline__ half8_t turned(half_t *tile, half8_t old, const float4_t (&o)[2], float factor)
{
    half8_t v = zero8();
    in_order();
    if constexpr (BASE) {
        put8(as_memory(tile), old);
        in_order();
        v = load8(as_operand(tile));
    }
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = f2h(BASE ? __builtin_fmaf(factor, o[e / 4][e % 4], h2f(v[e])) : factor * o[e / 4][e % 4]);
    in_order();
    put8(as_operand(tile), v);
    in_order();
    return load8(as_memory(tile));
}

// 32 columns of y for 16 TB rows whose h is in LDS: 32 rows of B, in an order that leaves a lane 8 columns side by side.
// lds: kLds halves, the wave's own.
template <int RT, int TB, bool BASE>
struct Columns {
    typedef Terms<RT> H;
    static constexpr int kLds = kTileHalves + 32 * (16 * RT + 8);
    half8_t w[RT], old[TB];
    int n0;
    __device__ __forceinline__ void load(const AdapterArgs &g, const Tile &t, const half_t *B, int n)
    {
        n0 = n;
        const int last = g.N * (g.R / 8) - 1;  // (rows of B are contiguous)
#pragma unroll
        for (int i = 0; i < RT; i++) w[i] = load8(B + 8 * (int64_t)min(n0 * (g.R / 8) + min(64 * i + (int)(threadIdx.x & 63), 4 * g.R - 1), last));
        if constexpr (BASE)
#pragma unroll
            for (int b = 0; b < TB; b++)
                old[b] = load8(g.base + (int64_t)(t.row0 + min(16 * b + mem_row(), t.rows - 1)) * g.ldb + min(n0 + mem_col(), g.N - 8));
    }
    __device__ __forceinline__ void put(const AdapterArgs &g, const Tile &t, const float (&factor)[TB], const half_t *hs, half_t *lds)
    {
        const int lane = threadIdx.x & 63, m = lane & 15, q4 = lane >> 4, per = g.R / 8, pitch = g.R + 8;
        half_t *const tile = lds, *const bl = lds + kTileHalves;
        in_order();
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int piece = min(64 * i + lane, 4 * g.R - 1);       // (as it was loaded: behind the last the last again)
            put8(bl + (piece / per) * pitch + 8 * (piece % per), w[i]);
        }
        if constexpr (BASE)
#pragma unroll
            for (int b = 0; b < TB; b++) arrived(old[b]);
        in_order();
        half8_t wf[2][H::kN];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < H::kN; i++) {
                wf[j][i] = load8(bl + (8 * (m >> 2) + 4 * j + (m & 3)) * pitch + min(H::of(i, q4), g.R - 8));
                wf[j][i] = H::of(i, q4) < g.R ? wf[j][i] : zero8();
            }
#pragma unroll
        for (int b = 0; b < TB; b++) {
            if (b && 16 * b >= t.rows) break;
            float4_t o[2] = {zero4(), zero4()};
#pragma unroll
            for (int i = 0; i < H::kN; i++)
#pragma unroll
                for (int p = 0; p < H::kM; p++) {
                    const half8_t hf = load8(hs + (16 * b + m) * H::kPitch + H::column(i, p, q4));
#pragma unroll
                    for (int j = 0; j < 2; j++) o[j] = mfma(wf[j][i], hf, o[j]);
                }
            const half8_t v = turned<BASE>(tile, old[b], o, factor[b]);
            const int r = 16 * b + mem_row(), c = n0 + mem_col();
            if (r < t.rows && c < g.N) *reinterpret_cast<half8_t *>(g.y + (int64_t)(t.row0 + r) * g.ldy + c) = v;
        }
    }
};
// The columns of a wave: those from 32 first on, every `stride`-th 32, each block's operands loaded when the last is done (the next ones' under way beside
// it cost registers: 2227 rows of 3200 to 8640, R = 64 34.2 us, 32.7 without)
template <int RT, int TB, bool BASE>
struct Wave {
    typedef Columns<RT, TB, BASE> C;
    const AdapterArgs &g;
    const Tile &t;
    const half_t *B;
    int n, step;
    C a;
    __device__ __forceinline__ Wave(const AdapterArgs &g_, const Tile &t_, int first, int stride) : g(g_), t(t_), n(32 * first), step(32 * stride)
    {
        B = g.B + (int64_t)t.a * g.N * g.R;
        a.load(g, t, B, n);
    }
    // largest: bits of the largest of each row of h
    __device__ __forceinline__ void run(float scale, const half_t *hs, const int *largest, half_t *lds)
    {
        if (n >= g.N) return;
        float factor[TB];
#pragma unroll
        for (int i = 0; i < TB; i++) factor[i] = factor_of(scale, exponent(largest[16 * i + (threadIdx.x & 15)]));
        for (;;) {
            a.put(g, t, factor, hs, lds);
            n += step;
            if (n >= g.N) break;
            a.load(g, t, B, n);
        }
    }
};

// rows without an adapter: the base, or nothing; of / splits of the work, by a workgroup
__device__ __forceinline__ void put_base(const AdapterArgs &g, const Tile &t, int of, int splits)
{
    if (of == 0)
        for (int e = threadIdx.x; e < t.rows * g.R; e += blockDim.x) g.h[(int64_t)t.row0 * g.R + e] = 0.f;
    if (g.base == g.y) return;
    for (int e = of * blockDim.x + threadIdx.x; e < t.rows * (g.N / 8); e += splits * blockDim.x) {
        const int64_t r = t.row0 + e / (g.N / 8);
        const int c = 8 * (e % (g.N / 8));
        *reinterpret_cast<half8_t *>(g.y + r * g.ldy + c) = g.base ? load8(g.base + r * g.ldb + c) : zero8();
    }
}

// Unit and split of a workgroup: the splits of a unit 8 apart, on one XCD, as they read the same
__device__ __forceinline__ int unit_and_split(const AdapterArgs &g, int *split)
{
    const int group = blockIdx.x / (8 * g.splits), left = min(8, (int)g.units.count - 8 * group);
    const int in = (int)blockIdx.x - 8 * group * g.splits;
    *split = in / left;
    return 8 * group + in % left;
}

// In one launch: a workgroup to 16 rows of a sequence and 1 / splits of the columns of y; h is formed by each of them.
constexpr int one_waves(int RT) { return RT <= 2 ? 16 : 8; }      // (the registers of more leave room for 8)
template <int RT, bool BASE>
__global__ void __launch_bounds__(64 * one_waves(RT)) one_kernel(AdapterArgs g)
{
    constexpr int W = one_waves(RT), C = 16 * RT;
    typedef TileH<RT, 1, W, false> H;
    typedef Wave<RT, 1, BASE> Y;
    typedef Terms<RT> Two;
    constexpr int kLds = std::max(std::max(W * H::kLds, 2 * W * kTile * C), W * Y::C::kLds);
    __shared__ __attribute__((aligned(16))) half_t lds[kLds], hs[kTile * Two::kPitch];
    __shared__ int largest[kTile];
    if ((int)blockIdx.x >= (int)g.units.count * g.splits) return look_over(g);
    int split;
    const int u = unit_and_split(g, &split);
    const Tile t = find_tile(g, u, kTile);
    if (t.rows == 0) return;
    if (t.a < 0) return put_base(g, t, split, g.splits);
    const float scale = g.scale[t.a];
    // (the first columns' operands are on their way before h is there)
    Y y(g, t, split * W + wave_id(), W * g.splits);
    H h(g.x + t.row0 * g.ldx, g.ldx, t.rows, g.K, g.A + (int64_t)t.a * g.R * g.K, g.R, lds + wave_id() * H::kLds);
    h.run(0, (g.K + 31) / 32);
    Two::clear(hs, kTile);
    if (threadIdx.x < kTile) largest[threadIdx.x] = 0;
    float sum[H::kItems];
    h.join(reinterpret_cast<float *>(lds), [&](int i, int r, int c, float s) __attribute__((always_inline)) {
        sum[i] = s;
        if (c >= g.R) return;
        atomicMax(largest + r, finite_bits(s));
        if (split == 0 && r < t.rows) g.h[(int64_t)(t.row0 + r) * g.R + c] = s;
    });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < H::kItems; i++) {
        const int e = threadIdx.x + 64 * W * i, r = e / C, c = e % C;
        if (e < kTile * C && c < g.R) Two::put(hs + r * Two::kPitch, c, sum[i] * two_to(-exponent(largest[r])));
    }
    __syncthreads();
    y.run(scale, hs, largest, lds + wave_id() * Y::C::kLds);
}

// In two, h first: 16 TB rows of a sequence and 1 / splits of the contraction to a workgroup, sums to a plane of [splits][T, R]
constexpr int kHBlocks = 2;
template <int RT, int TB>
__global__ void __launch_bounds__(512) h_kernel(AdapterArgs g, float *planes)
{
    constexpr int WAVES = 8;
    typedef TileH<RT, TB, WAVES, false> H;
    __shared__ __attribute__((aligned(16))) half_t lds[std::max(WAVES * H::kLds, 2 * WAVES * 16 * TB * 16 * RT)];
    if ((int)blockIdx.x >= (int)g.units.count * g.splits) return look_over(g);
    int split;
    const int u = unit_and_split(g, &split);
    const Tile t = find_tile(g, u, 16 * TB);
    if (t.rows == 0 || t.a < 0) return;
    H h(g.x + t.row0 * g.ldx, g.ldx, t.rows, g.K, g.A + (int64_t)t.a * g.R * g.K, g.R, lds + wave_id() * H::kLds);
    const int steps = (g.K + 31) / 32;
    h.run(steps * split / g.splits, steps * (split + 1) / g.splits);
    h.join(reinterpret_cast<float *>(lds), [&](int, int r, int c, float s) __attribute__((always_inline)) {
        if (c < g.R && r < t.rows) planes[((int64_t)split * g.pb.T + t.row0 + r) * g.R + c] = s;
    });
}

// .. then y: 64 rows and 1 / splits of the columns to a workgroup
constexpr int kRows = 64;
template <int RT, bool BASE>
__global__ void __launch_bounds__(512) y_kernel(AdapterArgs g, const float *planes, int count)
{
    constexpr int W = 8, NI = (RT + 1) / 2;
    typedef Terms<RT> Two;
    typedef Wave<RT, kRows / 16, BASE> Y;
    __shared__ __attribute__((aligned(16))) half_t hs[kRows * Two::kPitch], lds[W * Y::C::kLds];
    __shared__ int largest[kRows];
    int split;
    const int u = unit_and_split(g, &split);
    const Tile t = find_tile(g, u, kRows);
    if (t.rows == 0) return;
    if (t.a < 0) return put_base(g, t, split, g.splits);
    const float scale = g.scale[t.a];
    const int R = g.R;
    Y y(g, t, split * W + wave_id(), W * g.splits);
    Two::clear(hs, kRows);
    if (threadIdx.x < kRows) largest[threadIdx.x] = 0;
    float4_t v[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int e = threadIdx.x + 64 * W * i, r = min(e / (R / 4), t.rows - 1), c = 4 * (e % (R / 4));
        const int64_t at = (int64_t)(t.row0 + r) * R + c;
        v[i] = *reinterpret_cast<const float4_t *>(planes + at);
        for (int q = 1; q < count; q++) v[i] += *reinterpret_cast<const float4_t *>(planes + q * (int64_t)g.pb.T * R + at);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int e = threadIdx.x + 64 * W * i, r = e / (R / 4), c = 4 * (e % (R / 4));
        if (r >= t.rows) break;
        if (split == 0 && count > 1) *reinterpret_cast<float4_t *>(g.h + (int64_t)(t.row0 + r) * R + c) = v[i];
        atomicMax(largest + r, max(max(finite_bits(v[i][0]), finite_bits(v[i][1])), max(finite_bits(v[i][2]), finite_bits(v[i][3]))));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int e = threadIdx.x + 64 * W * i, r = e / (R / 4), c = 4 * (e % (R / 4));
        if (r >= t.rows) break;
        const float own = two_to(-exponent(largest[r]));
#pragma unroll
        for (int k = 0; k < 4; k++) Two::put(hs + r * Two::kPitch, c + k, v[i][k] * own);
    }
    __syncthreads();
    y.run(scale, hs, largest, lds + wave_id() * Y::C::kLds);
}

// ---------------------------------------------------------------- gradients
constexpr int kCols = 128;                     // (and kRows rows) of a step of the second kernel

struct GradArgs {
    AdapterArgs f;                             // x, A, B, h as in the forward pass; y, ldy: dx; base: what it is added to, or null
    const half_t *dy;
    int64_t lddy;
    half_t *terms[2];                          // of dh (without the scale) and h: rows of 32 RT, as in LDS, scaled by
    int *exps[2];                              // powers of two of their own
    int *rows, *begin;                         // rows of adapter a: rows[begin[a]] .. rows[begin[a + 1] - 1]
    int *part;                                 // the first part of adapter a, which has parts where it has several blocks
    float *parts;                              // of dA [R, K] and dB [N, R], a block of rows each
    half_t *dA, *dB;
    int dA_acc, dB_acc, per;                   // rows of a block
    int64_t blocks;
};

// The rows of each adapter, sequence after sequence, by one workgroup of 8 waves: each of up to 8 counts the rows of its share of the
// sequences by adapter (room: ints of LDS), then gives them their places, 64 sequences at a time.  (Sums no larger than T: sequences that
// overlap may have more rows than there are.  300 sequences of 300 adapters, each adapter looking through them all: 111 us.)
constexpr int kMaxAdapters = 1024;            // (the forward call takes no more than its adjoint)
__device__ void plan(const GradArgs &d, int *room, int ints, int *totals)
{
    const AdapterArgs &g = d.f;
    const int lane = threadIdx.x & 63, wave = wave_id(), T = g.pb.T, B = g.pb.B, shares = max(1, min(8, min(ints / g.n, B)));
    int *const own = room + wave * g.n;
    auto add = [&](int x, int y) __attribute__((always_inline)) { return min(x + y, T); };
    auto each = [&](auto f) __attribute__((always_inline)) {     // f(adapter or -1, first row, rows, sequences)
        if (wave >= shares) return;
        const int end = B * (wave + 1) / shares;
        for (int b0 = B * wave / shares; b0 < end; b0 += 64) {
            const int b = b0 + lane;
            int s0 = 0, n = 0;
            const bool there = rows_of(g, min(b, end - 1), &s0, &n) && b < end && n > 0;
            f(there ? adapter_of(g, b) : -1, s0, n, min(64, end - b0));
        }
    };
    auto count = [&](int a, int n) __attribute__((always_inline)) {
        if (a < 0) return;
        atomicAdd(own + a, n);                 // (64 of 2^24 and what was there: within 32 bits)
        atomicMin(own + a, T);
    };
    for (int e = threadIdx.x; e < shares * g.n; e += 512) room[e] = 0;
    __syncthreads();
    each([&](int a, int, int n, int) __attribute__((always_inline)) { count(a, n); });
    __syncthreads();
    // two adapters to a thread: where their rows begin
    const int a0 = 2 * (int)threadIdx.x;
    int mine[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; i++)
        for (int s = 0; s < shares && a0 + i < g.n; s++) mine[i] = add(mine[i], room[s * g.n + a0 + i]);
    auto before_this = [&](int v, auto plus) __attribute__((always_inline)) {      // of the threads before this one
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(v, o);
            if (lane >= o) v = plus(v, x);
        }
        if (lane == 63) totals[wave] = v;
        v = __shfl_up(v, 1);
        if (lane == 0) v = 0;
        __syncthreads();
        for (int w = 0; w < wave; w++) v = plus(v, totals[w]);
        __syncthreads();
        return v;
    };
    int before = before_this(add(mine[0], mine[1]), add), parts[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (a0 + i >= g.n) break;
        d.begin[a0 + i] = before;
        const int first = before;
        int at = before;
        for (int s = 0; s < shares; s++) {
            const int c = room[s * g.n + a0 + i];
            room[s * g.n + a0 + i] = at;
            at = add(at, c);
        }
        before = at;
        if (a0 + i == g.n - 1) d.begin[g.n] = at;
        parts[i] = at - first > d.per ? (at - first + d.per - 1) / d.per : 0;
    }
    const int part = before_this(parts[0] + parts[1], [](int x, int y) { return x + y; });
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (a0 + i < g.n) d.part[a0 + i] = part + (i ? parts[0] : 0);
    each([&](int a, int s0, int n, int sequences) __attribute__((always_inline)) {
        int at = a >= 0 ? own[a] : T;
        for (int l = 0; l < sequences; l++) {
            const int al = __builtin_amdgcn_readlane(a, l), nl = __builtin_amdgcn_readlane(n, l);
            if (l < lane && al == a) at = add(at, nl);
        }
        count(a, n);
        uint64_t todo = __ballot(a >= 0);
        while (todo) {
            const int l = __builtin_ctzll(todo);
            todo &= todo - 1;
            const int first = __builtin_amdgcn_readlane(s0, l), rows = __builtin_amdgcn_readlane(n, l), to = __builtin_amdgcn_readlane(at, l);
            for (int i = lane; i < rows && to + i < T; i += 64) d.rows[to + i] = first + i;
        }
    });
}

// The two terms of dh and h of 16 rows of a sequence; dx of rows without an adapter.  The first workgroup: the plan, the last: what does not fit.
template <int RT>
__global__ void __launch_bounds__(512) dh_kernel(GradArgs d)
{
    constexpr int W = 8, C = 16 * RT;
    typedef TileH<RT, 1, W, true> H;
    typedef Terms<RT> Two;
    __shared__ __attribute__((aligned(16))) half_t lds[std::max(W * H::kLds, 2 * W * kTile * C)], hs[kTile * Two::kPitch];
    __shared__ int largest[2][kTile];
    static_assert(sizeof(lds) / 4 >= kMaxAdapters && 2 * 512 >= kMaxAdapters, "room for a count, a thread for two");
    const AdapterArgs &g = d.f;
    if (blockIdx.x == 0) return plan(d, reinterpret_cast<int *>(lds), (int)sizeof(lds) / 4, largest[0]);
    const int u = (int)blockIdx.x - 1;
    if (u >= (int)g.units.count) return look_over(g);
    const Tile t = find_tile(g, u, kTile);
    if (t.rows == 0) return;
    const int R = g.R, K = g.K;
    if (t.a < 0) {
        if (g.base) return;                    // (added to: nothing)
        for (int e = threadIdx.x; e < t.rows * (K / 8); e += 64 * W)
            *reinterpret_cast<half8_t *>(g.y + (int64_t)(t.row0 + e / (K / 8)) * g.ldy + 8 * (e % (K / 8))) = zero8();
        return;
    }
    float sum[2][H::kItems];
#pragma unroll
    for (int i = 0; i < H::kItems; i++) {
        const int e = threadIdx.x + 64 * W * i, r = min(e / C, t.rows - 1), c = min(e % C, R - 1);
        sum[1][i] = g.h[(int64_t)(t.row0 + r) * R + c];
    }
    H h(d.dy + t.row0 * d.lddy, d.lddy, t.rows, g.N, g.B + (int64_t)t.a * g.N * R, R, lds + wave_id() * H::kLds);
    h.run(0, (g.N + 31) / 32);
    if (threadIdx.x < 2 * kTile) largest[threadIdx.x / kTile][threadIdx.x % kTile] = 0;
    h.join(reinterpret_cast<float *>(lds), [&](int i, int r, int c, float s) __attribute__((always_inline)) {
        sum[0][i] = s;
        if (c >= R) return;
        atomicMax(&largest[0][r], finite_bits(s));
        atomicMax(&largest[1][r], finite_bits(sum[1][i]));
    });
#pragma unroll
    for (int of = 0; of < 2; of++) {
        __syncthreads();
        Two::clear(hs, kTile);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < H::kItems; i++) {
            const int e = threadIdx.x + 64 * W * i, r = e / C, c = e % C;
            if (e < kTile * C && c < R) Two::put(hs + r * Two::kPitch, c, sum[of][i] * two_to(-exponent(largest[of][r])));
        }
        __syncthreads();
        for (int e = threadIdx.x; e < t.rows * 4 * RT; e += 64 * W)
            put8(d.terms[of] + ((int64_t)t.row0 * 4 * RT + e) * 8, load8(hs + e / (4 * RT) * Two::kPitch + 8 * (e % (4 * RT))));
        if ((int)threadIdx.x < t.rows) d.exps[of][t.row0 + threadIdx.x] = exponent(largest[of][threadIdx.x]);
    }
}

// units of adapter a begin at begin[a] / per + a
__device__ __forceinline__ int64_t unit_of(const GradArgs &d, int a) { return (int64_t)(d.begin[a] / d.per) + a; }

// A block of an adapter's rows and 128 columns: of x, for dx and the block's part of dA, or of dy, for its part of dB.  64 rows at a time
// in LDS, the next ones under way.
constexpr int kMostRows = 512;                 // of a block
template <int RT>
struct GradLds {
    static constexpr int HP = Terms<RT>::kPitch, XP = kCols + 16;
    // (A is in registers before the first rows come)
    __attribute__((aligned(16))) half_t rows_and_terms[std::max(kRows * (XP + HP), 16 * RT * XP)], tiles[4][kTileHalves], less[4][kRows];
    int exps[2][kRows], rows[kMostRows];
};
// rows first .. first + count - 1 of those of adapter a, its block `block`; columns from c0 on of x (and dx) or of dy.  (Either by itself: the operands of the
// sums change places, and the compiler makes a branch at each instruction of one that does both.)
template <int RT, bool of_x>
__device__ __forceinline__ void grad(const GradArgs &d, GradLds<RT> &l, int block, int a, int first, int count, int c0)
{
    typedef Terms<RT> Two;
    constexpr int HP = GradLds<RT>::HP, XP = GradLds<RT>::XP, NX = kRows * kCols / 8 / 256;
    half_t *const xs = l.rows_and_terms, *const hs = xs + kRows * XP, *const as = xs;
    auto &tiles = l.tiles;
    auto &less = l.less;
    auto &exps = l.exps;
    auto &rows = l.rows;
    const AdapterArgs &g = d.f;
    const int R = g.R, K = g.K, N = g.N, width = of_x ? K : N;
    const int lane = threadIdx.x & 63, wave = wave_id(), m = lane & 15, q4 = lane >> 4;
    const float scale = g.scale[a];
    const half_t *src = of_x ? g.x : d.dy, *terms = d.terms[of_x ? 0 : 1];
    const int64_t ld = of_x ? g.ldx : d.lddy;
    const int *from_exps = d.exps[of_x ? 0 : 1];
    for (int e = threadIdx.x; e < count; e += 256) rows[e] = d.rows[first + e];
    if constexpr (of_x)
        for (int e = threadIdx.x; e < 16 * RT * (kCols / 8); e += 256) {
            const int r = e / (kCols / 8), c = 8 * (e % (kCols / 8));
            const half8_t w = load8(g.A + ((int64_t)a * R + min(r, R - 1)) * K + min(c0 + c, K - 8));
            put8(as + r * XP + c, r < R && c0 + c < K ? w : zero8());
        }
    __syncthreads();
    half8_t x[NX], v[RT];
    int exp;
    const int xc = 8 * (threadIdx.x % (kCols / 8)), xr = threadIdx.x / (kCols / 8), vc = 8 * (threadIdx.x % (4 * RT)), vr = threadIdx.x / (4 * RT);
    auto load = [&](int r0) __attribute__((always_inline)) {      // (rows that there are not: others)
#pragma unroll
        for (int i = 0; i < NX; i++) x[i] = load8(src + (int64_t)rows[min(r0 + xr + 256 / (kCols / 8) * i, count - 1)] * ld + min(c0 + xc, width - 8));
#pragma unroll
        for (int i = 0; i < RT; i++) v[i] = load8(terms + (int64_t)rows[min(r0 + vr + 64 / RT * i, count - 1)] * (32 * RT) + vc);
        exp = from_exps[rows[min(r0 + lane, count - 1)]];
    };
    load(0);
    // A of 32 columns a wave, 8 of them side by side in a lane
    half8_t w[Two::kN][2];
    if constexpr (of_x)
#pragma unroll
    for (int i = 0; i < Two::kN; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const half_t *q = as + (Two::of(i, q4) + (m >> 2)) * XP + 32 * wave + 8 * (m & 3) + 4 * j;
            w[i][j] = both(read_tr(q), read_tr(q + 4 * XP));
        }
    __syncthreads();
    float4_t acc[RT][2];
#pragma unroll
    for (int i = 0; i < RT; i++) acc[i][0] = acc[i][1] = zero4();
    int top = -127;                            // exponent that the sums are scaled by
    // the sums over rows: step s has rows 32 s + 4 q4 + 0 .. 3 and those 16 further, in both operands
    auto sums = [&] () __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < kRows / 32; s++) {
            const int row = 32 * s + 4 * q4 + (m >> 2);
            const half_t *f = less[wave] + 32 * s + 4 * q4;
            const half8_t part = both(*reinterpret_cast<const half4_t *>(f), *reinterpret_cast<const half4_t *>(f + 16));
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
                    const half_t *q = hs + row * HP + p * Two::kLo + 16 * i + 4 * (m & 3);
                    const half8_t hf = both(read_tr(q), read_tr(q + 16 * HP)) * part;
#pragma unroll
                    for (int c = 0; c < 2; c++) acc[i][c] = of_x ? mfma(hf, xf[c], acc[i][c]) : mfma(xf[c], hf, acc[i][c]);
                }
        }
    };
    for (int r0 = 0, turn = 0; r0 < count; r0 += kRows, turn ^= 1) {
        const int left = count - r0;
#pragma unroll
        for (int i = 0; i < NX; i++) {
            const int r = xr + 256 / (kCols / 8) * i;
            put8(xs + r * XP + xc, r < left && c0 + xc < width ? x[i] : zero8());
        }
#pragma unroll
        for (int i = 0; i < RT; i++) {
            const int r = vr + 64 / RT * i;
            put8(hs + r * HP + vc, r < left ? v[i] : zero8());
        }
        // rows' scales, as parts of the largest so far: one below 2^-24 of it is lost
        if (lane >= left) exp = -127;
        const int now = max(top, (int)wave_max((float)exp));
        less[wave][lane] = f2h(two_to(max(exp - now, -126)));
        if (wave == 0) exps[turn][lane] = exp;
        if (now > top) {
            const float f = two_to(max(top - now, -126));
            top = now;
#pragma unroll
            for (int i = 0; i < RT; i++) acc[i][0] *= f, acc[i][1] *= f;
        }
        // (what dx is added to: before the next rows, which the wait for it would be one for too)
        half8_t old[kRows / 16];
        if constexpr (of_x)
            if (g.base)
#pragma unroll
                for (int t = 0; t < kRows / 16; t++)
                    old[t] = load8(g.base + (int64_t)rows[r0 + min(16 * t + mem_row(), left - 1)] * g.ldb + min(c0 + 32 * wave + mem_col(), K - 8));
        load(r0 + kRows);
        __syncthreads();
        sums();
        if constexpr (of_x)
#pragma unroll
            for (int t = 0; t < kRows / 16; t++) {
                if (16 * t >= left) break;
                float4_t o[2] = {zero4(), zero4()};
#pragma unroll
                for (int i = 0; i < Two::kN; i++)
#pragma unroll
                    for (int p = 0; p < Two::kM; p++) {
                        const half8_t hf = load8(hs + (16 * t + m) * HP + Two::column(i, p, q4));
#pragma unroll
                        for (int j = 0; j < 2; j++) o[j] = mfma(w[i][j], hf, o[j]);
                    }
                const float factor = factor_of(scale, exps[turn][16 * t + m]);
                const int r = 16 * t + mem_row(), c = c0 + 32 * wave + mem_col();
                const int64_t row = rows[r0 + min(r, left - 1)];
                half8_t y;
                if (g.base) y = turned<true>(tiles[wave], old[t], o, factor);
                else y = turned<false>(tiles[wave], zero8(), o, factor);
                if (r < left && c < K) *reinterpret_cast<half8_t *>(g.y + row * g.ldy + c) = y;
            }
        __syncthreads();
    }
    const float up = two_to(max(top, -126));
    const bool alone = d.begin[a + 1] - d.begin[a] <= d.per;      // (the only block: nothing to be joined)
    const int64_t ofA = (int64_t)R * K, ofB = (int64_t)R * N;
    float *const part = d.parts + (int64_t)(d.part[a] + block) * (ofA + ofB) + (of_x ? 0 : ofA);
    half_t *const to = of_x ? d.dA + a * ofA : d.dB + a * ofB;
    const bool add = of_x ? d.dA_acc : d.dB_acc;
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int r = 16 * i + (of_x ? 4 * q4 + e : m), col = c0 + 32 * wave + 16 * c + (of_x ? m : 4 * q4 + e);
                if (r >= R || col >= width) continue;
                const int64_t at = of_x ? (int64_t)r * K + col : (int64_t)col * R + r;
                const float v = up * acc[i][c][e];
                if (alone) to[at] = add ? f2h(h2f(to[at]) + scale * v) : f2h(scale * v);
                else part[at] = v;
            }
}

template <int RT>
__global__ void __launch_bounds__(256, RT == 8 ? 2 : RT == 4 ? 3 : 4) grad_kernel(GradArgs d)
{
    __shared__ GradLds<RT> l;
    // (x's columns, which take longer, before dy's)
    const int kchunks = (d.f.K + kCols - 1) / kCols, nchunks = (d.f.N + kCols - 1) / kCols, of_x = (int)d.blocks * kchunks;
    const bool x = (int)blockIdx.x < of_x;
    const int i = x ? (int)blockIdx.x : (int)blockIdx.x - of_x, u = i / (x ? kchunks : nchunks), chunk = i - u * (x ? kchunks : nchunks);
    // (unit 0 is adapter 0's: one more than the adapters that begin behind it)
    const int a = __builtin_amdgcn_readfirstlane(count_below(d.f.n - 1, u, [&](int i) { return unit_of(d, i); }));
    const int block = (int)(u - unit_of(d, a)), first = d.begin[a] + block * d.per, count = min(d.per, d.begin[a + 1] - first);
    if (count <= 0) return;
    if (x) grad<RT, true>(d, l, block, a, first, count, kCols * chunk);
    else grad<RT, false>(d, l, block, a, first, count, kCols * chunk);
}

// The parts of an adapter that has several blocks added up, and what has none made 0; 4 elements to a thread
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
    if (parts == 1 || (parts == 0 && acc)) return;
    const float *p = d.parts + (int64_t)d.part[a] * size + e;
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

// Memory that a call reads or writes, from its first element to its last, in halves
struct Extent {
    const void *at;
    int64_t size;
};
Extent rows_extent(int64_t T, const void *p, int64_t ld, int64_t width) { return {p, p ? (T - 1) * ld + width : 0}; }
bool share(const Extent &a, std::initializer_list<Extent> others)
{
    for (const Extent &b : others)
        if (b.size && rows_share(1, a.at, 0, a.size, b.at, 0, b.size)) return true;
    return false;
}

// RT of 1, 2, 4 or 8: R rounded up to 16 of them
int rank_of(int64_t R) { return R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8; }
#define CACTI_BY_RANK(R, launch)        \
    do {                                \
        if ((R) <= 16) launch(1);       \
        else if ((R) <= 32) launch(2);  \
        else if ((R) <= 64) launch(4);  \
        else launch(8);                 \
    } while (0)

// rows of a block: as many workgroups as the device holds at once, counting those of blocks that are not full.  (4096 rows of 3200 to 3200,
// R = 64: about 640 54 us, 768 57, 384 59; R = 128, two to a CU: 384 90, 640 101; before other steps that took 5 and 14 us off either.)
int64_t block_rows(int64_t T, int64_t K, int64_t N, int64_t R)
{
    const int64_t chunks = (K + kCols - 1) / kCols + (N + kCols - 1) / kCols, steps = (T + kRows - 1) / kRows;
    int64_t per = steps * chunks / (R > 64 ? 384 : 640);
    per = per < 1 ? 1 : per > kMostRows / kRows ? kMostRows / kRows : per;
    return per * kRows;
}

struct Workspace {
    size_t terms[2], exps[2], rows, begin, part, parts, bytes;
    int64_t per, blocks;
};
Workspace workspace(int64_t T, int64_t K, int64_t N, int64_t R, int64_t n)
{
    Workspace w;
    w.bytes = 0;
    auto room = [&](size_t b) {
        const size_t at = w.bytes;
        w.bytes += (b + 255) / 256 * 256;
        return at;
    };
    w.per = block_rows(T, K, N, R);
    w.blocks = T / w.per + n;
    for (int i = 0; i < 2; i++) {
        w.terms[i] = room((size_t)T * 64 * rank_of(R));
        w.exps[i] = room((size_t)T * 4);
    }
    w.rows = room((size_t)T * 4);
    w.begin = room((size_t)(n + 1) * 4);
    w.part = room((size_t)n * 4);
    // Parts are those of adapters with more than a block of rows: of c > per rows ceil(c / per) <= 2 c / (per + 1).  (With one for every adapter
    // 512 rows of 1024 adapters, 3200 to 8640, R = 128, took 6 GB.  There is room for one for each as long as that is no more than 32 MB.)
    const size_t size = (size_t)R * (K + N) * 4;
    const int64_t parts = std::min(2 * T / (w.per + 1), w.blocks), spare = std::min<int64_t>(n, (32 << 20) / size);
    w.parts = room(std::max(parts, spare) * size);
    return w;
}

// How the forward pass is cut: in one launch, whose workgroups of 16 rows each form the h that they need, over all of K, with the columns
// split until the device is full; or h first, from parts of K, and then y by 64 rows: a launch more, but A and B are read less often.  The
// second, by us of both (the second's first), where
//   K is long and A large, and the tiles leave half of the device idle: one row of 8640 to 3200, R = 32 10.6 and 13.3, R = 128 18.6 and 32.5,
//     1200 rows 33 and 52; not with K = 3200, whose 600 rows with R = 128 take 27.1 and 23.4;
//   there are rows for several rounds of tiles: 16 x 600 rows of 2048 to 2048, R = 8 27 and 29, R = 32 33 and 38, R = 128 67 and 80;
//   the tiles are too few to fill the device and too many to split their columns, and A and B are large: 4 x 557 rows of 3200 to 8640,
//     R = 64 33 and 45, but R = 16 23.3 either way.
// Everywhere else the first: one row of 3200 to 8640, R = 16 8.5 and 6.2, 2048 rows of 3200 to 3200 13.2 and 10.4, 4096 19.1 and 15.7.
// Over 125 shapes (profiles/adapter_forward_launches.txt) the rule's choice is 0.7 % slower than the better one in the mean, 13 % at most.  None of
// them has K between 3200 and 8640: that the border is 4096 there is a guess.
struct ForwardPlan {
    bool two;
    int splits, planes;
    Units h_units, y_units;
    size_t bytes;
};
ForwardPlan forward_plan(int64_t T, int64_t S, int64_t K, int64_t N, int64_t R, int64_t max_new)
{
    ForwardPlan w{};
    auto units = [&](int64_t rows) { return make_units(T, S, rows, 1, 1, (max_new + rows - 1) / rows); };
    auto fill = [](int64_t target, int64_t count, int64_t most) { return (int)std::max<int64_t>(1, std::min(target / count, most)); };
    // splits of the columns among workgroups of some waves: no more than give the busiest wave fewer
    auto columns = [&](int64_t target, int64_t count, int64_t waves) {
        const int64_t blocks = (N + 31) / 32, most = fill(target, count, (blocks + waves - 1) / waves), turns = (blocks + waves * most - 1) / (waves * most);
        return (int)((blocks + waves * turns - 1) / (waves * turns));
    };
    const int64_t cus = device_cus();
    const int rank = rank_of(R);
    const int64_t tiles = units(kTile).count;
    w.two = (K > 4096 && R * K > (1 << 18) && tiles <= cus / 2) || T >= 32 * cus ||
            (tiles > cus / 2 && tiles < cus && R * (K + N) > (1 << 18));
    if (!w.two) {
        w.splits = columns(cus, tiles, one_waves(rank));
        return w;
    }
    w.h_units = units(16 * kHBlocks);
    w.y_units = units(kRows);
    w.planes = fill(cus, w.h_units.count, std::min<int64_t>(8, (K + 255) / 256));
    w.splits = columns(rank == 8 ? cus : 2 * cus, w.y_units.count, 8);       // (as many as a CU's LDS has room for: R = 128 47 us, by two 54)
    w.bytes = w.planes > 1 ? (size_t)w.planes * T * R * 4 : 0;
    return w;
}

}  // namespace

CACTI_API size_t cacti_hip_adapter_fwd_workspace(int64_t T, int64_t S, int64_t K, int64_t N, int64_t R, int64_t max_new)
{
    return T > 0 && S > 0 && K > 0 && N > 0 && R > 0 && max_new > 0 ? forward_plan(T, S, K, N, R, max_new < T ? max_new : T).bytes : 0;
}

CACTI_API int cacti_hip_adapter_fwd(int64_t T, int64_t S, int64_t K, int64_t N, int64_t R, int64_t n, int64_t max_new, const void *x, int64_t ldx,
                                    const void *A, const void *B, const void *starts, const void *ids, const void *scale, const void *base,
                                    int64_t ldb, void *y, int64_t ldy, void *h, void *ws, size_t ws_bytes, void *status, void *stream)
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
    const ForwardPlan w = forward_plan(T, S, K, N, R, g.max_new);
    CACTI_REQUIRE(ws_bytes >= w.bytes && (ws || !w.bytes) && aligned(ws, 16), CACTI_E_INVALID, "adapter_fwd: workspace of %zu bytes, %zu needed, 16-byte aligned",
                  ws_bytes, w.bytes);
    // (some workgroups read while others write)
    const Extent eA = {A, n * R * K}, eB = {B, n * N * R}, eh = {h, 2 * T * R};
    CACTI_REQUIRE(!share(rows_extent(T, y, ldy, N), {eA, eB, eh}) && !share(eh, {rows_extent(T, x, ldx, K), rows_extent(T, base, ldb, N), eA, eB}), CACTI_E_INVALID,
                  "adapter_fwd: y or h shares memory with an operand or the other");
    hipStream_t st = (hipStream_t)stream;
    if (!w.two) {
        g.splits = w.splits;
        const int64_t blocks = g.units.count * g.splits + (status ? 1 : 0);
        CACTI_REQUIRE(blocks <= INT32_MAX, CACTI_E_NOTIMPL, "adapter_fwd: too many tiles");
#define LAUNCH(RT)                                                                                                       \
    do {                                                                                                                 \
        if (base) hipLaunchKernelGGL((one_kernel<RT, true>), dim3((unsigned)blocks), dim3(64 * one_waves(RT)), 0, st, g); \
        else hipLaunchKernelGGL((one_kernel<RT, false>), dim3((unsigned)blocks), dim3(64 * one_waves(RT)), 0, st, g);     \
    } while (0)
        CACTI_BY_RANK(R, LAUNCH);
#undef LAUNCH
        return launch_status("adapter_fwd");
    }
    float *planes = w.planes > 1 ? (float *)ws : g.h;
    AdapterArgs first = g;
    first.units = w.h_units;
    first.splits = w.planes;
    g.units = w.y_units;
    g.splits = w.splits;
    const int64_t blocks1 = first.units.count * first.splits + (status ? 1 : 0), blocks2 = g.units.count * g.splits;
    CACTI_REQUIRE(blocks1 <= INT32_MAX && blocks2 <= INT32_MAX, CACTI_E_NOTIMPL, "adapter_fwd: too many tiles");
#define LAUNCH(RT)                                                                                                       \
    do {                                                                                                                 \
        hipLaunchKernelGGL((h_kernel<RT, kHBlocks>), dim3((unsigned)blocks1), dim3(512), 0, st, first, planes);                     \
        if (base) hipLaunchKernelGGL((y_kernel<RT, true>), dim3((unsigned)blocks2), dim3(512), 0, st, g, (const float *)planes, w.planes); \
        else hipLaunchKernelGGL((y_kernel<RT, false>), dim3((unsigned)blocks2), dim3(512), 0, st, g, (const float *)planes, w.planes);     \
    } while (0)
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
    CACTI_REQUIRE(!rows_share(1, dA, n * R * K, n * R * K, dB, n * N * R, n * N * R), CACTI_E_INVALID, "adapter_bwd: dA shares memory with dB");
    const Workspace w = workspace(T, K, N, R, n);
    CACTI_REQUIRE(ws_bytes >= w.bytes, CACTI_E_INVALID, "adapter_bwd: workspace of %zu bytes, %zu needed", ws_bytes, w.bytes);
    const int64_t chunks = (K + kCols - 1) / kCols + (N + kCols - 1) / kCols, size = R * (K + N);
    CACTI_REQUIRE(w.blocks * chunks < (1 << 24), CACTI_E_NOTIMPL, "adapter_bwd: too many tiles");
    // (an adapter's gradient is written while others are formed)
    const Extent eA = {A, n * R * K}, eB = {B, n * N * R}, eh = {h, 2 * T * R}, edx = rows_extent(T, dx, lddx, K);
    CACTI_REQUIRE(!share(edx, {eA, eB, eh}), CACTI_E_INVALID, "adapter_bwd: dx shares memory with A, B or h");
    const Extent ex = rows_extent(T, x, ldx, K), edy = rows_extent(T, dy, lddy, N);
    CACTI_REQUIRE(!share({dA, eA.size}, {ex, edy, edx, eA, eB, eh}) && !share({dB, eB.size}, {ex, edy, edx, eA, eB, eh}), CACTI_E_INVALID,
                  "adapter_bwd: dA or dB shares memory with an operand or dx");
    char *p = (char *)ws;
    d.f.h = (float *)const_cast<void *>(h);
    d.f.y = (half_t *)dx, d.f.ldy = lddx;
    d.f.base = dx_acc ? (const half_t *)dx : nullptr, d.f.ldb = lddx;
    d.dy = (const half_t *)dy, d.lddy = lddy;
    for (int i = 0; i < 2; i++) d.terms[i] = (half_t *)(p + w.terms[i]), d.exps[i] = (int *)(p + w.exps[i]);
    d.rows = (int *)(p + w.rows), d.begin = (int *)(p + w.begin), d.part = (int *)(p + w.part);
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
