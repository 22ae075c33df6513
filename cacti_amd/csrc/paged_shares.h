// How the work of a call of attention over a paged cache is cut (paged_attention.hip): tiles of rows, steps over their positions, equal
// shares of all steps to the workgroups, and the pages that a part of a tile looks up.  Whole numbers alone, the same on the host.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define CACTI_BOTH __host__ __device__ __forceinline__
#else
#define CACTI_BOTH inline
#endif

namespace cacti {
namespace shares {

template <class T>
CACTI_BOTH T lesser(T a, T b) { return b < a ? b : a; }
template <class T>
CACTI_BOTH T larger(T a, T b) { return a < b ? b : a; }

// What is the same in all lanes, in a scalar register
CACTI_BOTH int same(int x)
{
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_readfirstlane(x);
#else
    return x;
#endif
}

constexpr int kWaves = 4, kStep = 32;
constexpr int kEntries = 64;                   // pages that a wave looks up at a time, one to a lane

// x / page for x below kEntries pages
constexpr unsigned magic_of(int64_t page) { return (unsigned)((1 << 22) / page + 1); }
CACTI_BOTH int page_of(int x, unsigned magic)
{
#ifdef __HIP_DEVICE_COMPILE__
    return (int)(__umul24((unsigned)x, magic) >> 22);
#else
    return (int)((((unsigned)x & 0xffffffu) * (magic & 0xffffffu)) >> 22);
#endif
}

// The pages of a part of a tile from position `seg` on, up to its end c1 or as many as are looked up at once: p0 .. p0 + last of the
// sequence's row of the table; positions are counted from base, the first of page p0, up to end
struct Pages {
    int p0, base, end;
    CACTI_BOTH Pages(int seg, int c1, int page) : p0(seg / page), base(p0 * page), end(lesser(c1 - base, kEntries * page)) {}
    CACTI_BOTH int last(unsigned magic) const { return page_of(end - 1, magic); }
};

// Equal shares of `units`: group i has those from begin(i) to begin(i + 1), the first `more` of them one more than `each`
struct Shares {
    unsigned each, more;
    CACTI_BOTH Shares(unsigned units, unsigned groups) : each(units / groups), more(units - each * groups) {}
    CACTI_BOTH unsigned begin(unsigned i) const { return i * each + lesser(i, more); }
    CACTI_BOTH unsigned of(unsigned unit) const          // the group that has it
    {
        const unsigned edge = more * (each + 1);
        return unit < edge ? unit / (each + 1) : more + (unit - edge) / each;
    }
};

// What a tile of rows costs a share besides its steps, in steps: queries, pages and the first keys to wait for.  (48 sequences
// of 120 to 8192 positions, 16 rows, 1 / 2 / 4 / 8: 130.2 / 128.4 / 129.4 / 131.3 us; 24 of 100 to 6000, 32 rows, 2 / 4 / 8 / 16:
// 29.1 / 27.7 / 28.5 / 29.4)
constexpr int begin_of(int tile) { return tile / 8; }

// A wave's part of a share is at least that many units: fewer steps are more parts to put together than they save (one sequence of
// 1540 positions, 32 heads of 100, 1 / 2 / 3 / 4: 13.7 / 12.4 / 13.1 / 13.5 us)
constexpr unsigned kLeast = 2;
constexpr unsigned kBigLeast = 4;              // the same of steps of 64 positions, to a workgroup
CACTI_BOTH unsigned groups_of(unsigned most, unsigned units) { return lesser(most, larger(units / (kLeast * kWaves), 1u)); }
CACTI_BOTH unsigned big_groups_of(unsigned most, unsigned units) { return lesser(most, larger(units / kBigLeast, 1u)); }

// A sequence's share of the work: its tiles of rows (tokens by the G query heads of a key head) by its steps (and begin_of), by heads
struct Share {
    int tiles, steps;
    unsigned units;
    CACTI_BOTH Share(int tile, int rows, int len, int Hkv, bool counted)
        : tiles((rows + tile - 1) / tile), steps((len + kStep - 1) / kStep), units(counted ? (unsigned)(tiles * (steps + begin_of(tile)) * Hkv) : 0u)
    {
    }
};
// Of units x .. until - 1 of the work, x in this sequence (before it: `before` units), those of one tile: h, row0 which; steps u0 .. u1 - 1 of it to
// a wave, g0 .. g1 - 1 to its workgroup, whose units are x0 .. x1 - 1
struct Part {
    int h, row0;
    unsigned start, end, g0, g1, u0, u1;       // the tile's steps: start .. end - 1
    CACTI_BOTH Part(const Share &w, int tile, unsigned before, unsigned x, unsigned until, unsigned x0, unsigned x1)
    {
        const unsigned whole = w.steps + begin_of(tile);
        const int u = same((int)((x - before) / whole));
        start = before + u * whole + begin_of(tile);
        end = start + w.steps;
        h = same(u / w.tiles);
        row0 = (u - h * w.tiles) * tile;
        g0 = larger(x0, start), u0 = larger(x, start), u1 = lesser(until, end);
        g1 = lesser(x1, end);
    }
    // positions of the wave, of which some row sees the first `seen`
    CACTI_BOTH int c0() const { return (int)(u0 - start) * kStep; }
    CACTI_BOTH int c1(int seen) const { return lesser(seen, (int)(u1 - start) * kStep); }
    // where the workgroup's sums go: to the output, or to its first or second place for partial ones
    CACTI_BOTH int slot(unsigned group) const { return g0 == start && g1 == end ? -1 : 2 * (int)group + (g0 == start); }
};

// Prompts: tiles of 128 rows, steps of 64 positions.  A tile's steps grow by those of its own rows: counted by a line that is
// never below them, so that what lies before a tile is a formula; steps behind a tile's last position are nothing.
constexpr int kPrompt = 128, kBig = 64;
// As begin_of, in steps.  (Prompts of up to 900 rows and 4000 positions, 16 heads of 128, 2 / 3 / 4 / 5: 74.9 / 73.3 / 71.4 / 74.0 us; one
// of 4096 130 / 121 / 122 / 125)
constexpr int kBigBegin = 4;
struct BigShare {
    int tiles, base, slope, run;               // steps of tile t: base + slope (t + 1), or, slope 0, base + t / run + 1
    CACTI_BOTH BigShare(int G, int rows, int first, bool counted)
    {
        const int tokens = (kPrompt + G - 1) / G;
        tiles = counted ? (rows + kPrompt - 1) / kPrompt : 0;
        base = (first + kBig - 1) / kBig + kBigBegin;
        slope = tokens >= kBig ? (tokens + kBig - 1) / kBig : 0;
        run = slope ? 1 : kBig / tokens;
    }
    CACTI_BOTH unsigned before(int t) const      // tile t
    {
        if (slope) return (unsigned)(t * base + slope * (t * (t + 1) / 2));
        const int q = t / run, r = t - q * run;
        return (unsigned)(t * base + run * (q * (q - 1) / 2) + r * q + t);
    }
    CACTI_BOTH unsigned units(int Hkv) const { return before(tiles) * (unsigned)Hkv; }
};
// Of a tile of `whole` units those from `from` to `to` - 1, positions c0 .. c1 - 1 (none, c0 >= c1 > 0, where they are behind the
// `seen` that some row sees)
struct BigPart {
    int first, behind, whole;                  // steps first .. behind - 1; none: only the tile's begin
    CACTI_BOTH BigPart(int from, int to, int whole) : first(larger(from - kBigBegin, 0)), behind(to - kBigBegin), whole(whole - kBigBegin) {}
    CACTI_BOTH int c0() const { return first * kBig; }
    CACTI_BOTH int c1(int seen) const { return lesser(seen, behind * kBig); }
    CACTI_BOTH int slot(unsigned group) const { return first == 0 && behind == whole ? -1 : 2 * (int)group + (first == 0); }
    // from where pages are looked up first: a page that there is, also where there is nothing to do
    CACTI_BOTH static int look(int c0, int c1) { return lesser(c0, c1 - 1); }
};

// Where the parts of a tile are whose steps are units first .. first + steps - 1: those of its first step's group, of the next ones and
// of its last step's
struct Parts {
    int i0, count;
    CACTI_BOTH Parts(unsigned units, unsigned groups, unsigned first, unsigned steps)
    {
        const Shares s(units, groups);
        i0 = (int)s.of(first);
        count = (int)s.of(first + steps - 1) - i0 + 1;
    }
    CACTI_BOTH int slot(int p) const { return p == 0 ? 2 * i0 + 1 : 2 * (i0 + p); }
};

}  // namespace shares
}  // namespace cacti
