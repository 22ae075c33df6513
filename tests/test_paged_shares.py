"""How the work of an attention call over a paged cache is cut (csrc/paged_shares.h, which the kernels are built from and which has no
device code): compiled into a small program here that walks all shares of random batches as the kernels do.  Every tile has every
position that its rows see exactly once, the places of partial sums are those that the join reads, and no page is looked up beyond
those of the sequence, in a table that has no more."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cacti_amd", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include <stdlib.h>

#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "paged_shares.h"

using namespace cacti::shares;

#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); exit(1); } } while (0)

struct Seq { int n, first; };
typedef std::tuple<int, int, int> Tile;        // sequence, head, first row

struct Batch {
    std::vector<Seq> seqs;
    int G, Hkv, page, few, groups, big_groups;
    std::map<Tile, std::vector<std::pair<int, int>>> seen, big_seen;       // what was done of a tile
    std::map<Tile, std::vector<int>> slots, big_slots;

    int len(int b) const { return seqs[b].first + seqs[b].n; }
    Share share(int tile, int b) const { return Share(tile, seqs[b].n * G, len(b), Hkv, seqs[b].n > 0 && seqs[b].n * G <= few); }
    BigShare big(int b) const { return BigShare(G, seqs[b].n * G, seqs[b].first, seqs[b].n * G > few); }

    void look_up(int b, int seg, int c1) const
    {
        const unsigned magic = magic_of(page);
        const Pages p(seg, c1, page);
        const int last = p.last(magic);
        CHECK(p.p0 >= 0 && last >= 0 && last < kEntries && (p.p0 + last) * page < len(b));
        CHECK(p.base <= seg && p.end > seg - p.base && p.base + p.end <= c1);
        for (int x = 0; x < p.end; x += x % page ? page - 1 : 1) CHECK(page_of(x, magic) == x / page && x / page <= last);
    }
    void pages(int b, int c0, int c1) const
    {
        for (int seg = c0; seg < c1;) {
            look_up(b, seg, c1);
            const Pages p(seg, c1, page);
            seg = p.base + p.end;
        }
    }
    // the units before sequence b's, and the sequence that x lies in
    template <class F>
    int find(unsigned x, unsigned *before, F units) const
    {
        *before = 0;
        for (int b = 0; b < (int)seqs.size(); b++) {
            if (*before + units(b) > x) return b;
            *before += units(b);
        }
        CHECK(!"a unit of nobody's");
        return -1;
    }

    unsigned few_rows(int tile)
    {
        auto units_of = [&](int b) { return share(tile, b).units; };
        uint64_t all = 0;
        for (int b = 0; b < (int)seqs.size(); b++) all += units_of(b);
        CHECK(all < INT32_MAX);
        const unsigned units = (unsigned)all, n = groups_of(groups, units);
        const Shares shares(units, n);
        for (unsigned group = 0; group < n; group++) {
            const unsigned x0 = shares.begin(group), x1 = shares.begin(group + 1);
            auto begin = [&](unsigned w) { return x0 + (x1 - x0) * w / kWaves; };
            std::map<Tile, int> owners, parts;
            for (unsigned wid = 0; wid < kWaves; wid++) {
                unsigned x = begin(wid), before;
                const unsigned until = begin(wid + 1);
                if (x >= until) continue;
                for (int b = find(x, &before, units_of), deposits = 0; x < until; b++) {
                    const Share w = share(tile, b);
                    const unsigned behind = before + w.units;
                    while (x < until && x < behind) {
                        const Part p(w, tile, before, x, until, x0, x1);
                        const int rows = seqs[b].n * G;
                        CHECK(p.u1 > x && p.h >= 0 && p.h < Hkv && p.row0 >= 0 && p.row0 < rows);
                        x = p.u1;
                        if (p.u1 <= p.u0) continue;
                        const int sees = seqs[b].first + lesser(rows - 1, p.row0 + tile - 1) / G + 1, c0 = p.c0(), c1 = p.c1(sees);
                        const Tile t(b, p.h, p.row0);
                        if (c0 < c1) {
                            pages(b, c0, c1);
                            seen[t].push_back({c0, c1});
                        }
                        parts[t]++;
                        if (p.u0 > p.g0) {
                            CHECK(++deposits == 1 && wid > 0);                   // a wave has one place in LDS for them
                            CHECK(owners.count(t));
                        } else {
                            CHECK(!owners.count(t));
                            owners[t] = p.slot(group);
                            CHECK(p.u1 >= p.g1 || x >= until);                  // others' come only to its last tile
                        }
                    }
                    before = behind;
                }
            }
            for (auto &o : owners) slots[o.first].push_back(o.second);
            for (auto &o : parts) CHECK(owners.count(o.first));
        }
        return units;
    }

    unsigned prompts()
    {
        auto units_of = [&](int b) { return big(b).units(Hkv); };
        uint64_t all = 0;
        for (int b = 0; b < (int)seqs.size(); b++) all += units_of(b);
        CHECK(all < INT32_MAX);
        const unsigned units = (unsigned)all, n = big_groups_of(big_groups, units);
        if (units == 0) return 0;
        const Shares shares(units, n);
        for (unsigned group = 0; group < n; group++) {
            unsigned x = shares.begin(group), before;
            const unsigned until = shares.begin(group + 1);
            if (x >= until) continue;
            for (int b = find(x, &before, units_of); x < until; b++) {
                const BigShare w = big(b);
                const unsigned head = w.before(w.tiles), behind = before + w.units(Hkv);
                while (x < until && x < behind) {
                    const int h = (int)((x - before) / head), rows = seqs[b].n * G;
                    const unsigned in = x - before - h * head;
                    int tile = 0;
                    while (tile < w.tiles && w.before(tile + 1) <= in) tile++;
                    CHECK(h < Hkv && tile < w.tiles);
                    const unsigned start = w.before(tile), whole = w.before(tile + 1) - start;
                    const int from = (int)(in - start), to = (int)lesser(whole, from + (until - x)), row0 = tile * kPrompt;
                    const int end = seqs[b].first + lesser(rows - 1, row0 + kPrompt - 1) / G + 1;
                    const BigPart p(from, to, (int)whole);
                    if (p.behind > p.first) {
                        const int c0 = p.c0(), c1 = p.c1(end);
                        CHECK(c1 > 0 && c0 >= 0);
                        look_up(b, BigPart::look(c0, c1), c1);
                        if (c0 < c1) {
                            pages(b, c0, c1);
                            big_seen[Tile(b, h, row0)].push_back({c0, c1});
                        }
                        big_slots[Tile(b, h, row0)].push_back(p.slot(group));
                    }
                    CHECK(to > from);
                    x += to - from;
                }
                before = behind;
            }
        }
        return units;
    }

    void check(int tile)
    {
        const unsigned units = few_rows(tile), big_units = prompts();
        std::map<int, int> used, big_used;
        unsigned before = 0, big_before = 0;
        for (int b = 0; b < (int)seqs.size(); b++) {
            const bool prompt = seqs[b].n * G > few;
            const Share w = share(tile, b);
            const BigShare big_w = big(b);
            const int rows = seqs[b].n * G, size = prompt ? kPrompt : tile;
            for (int h = 0; h < Hkv; h++)
                for (int t = 0; t * size < rows; t++) {
                    const Tile at(b, h, t * size);
                    int upto = 0;              // (parts come in the order of their positions)
                    for (auto &c : (prompt ? big_seen : seen)[at]) {
                        CHECK(c.first == upto && c.second > c.first);
                        upto = c.second;
                    }
                    CHECK(upto == seqs[b].first + lesser(rows - 1, t * size + size - 1) / G + 1);
                    const unsigned first = prompt ? big_before + h * big_w.before(big_w.tiles) + big_w.before(t) + kBigBegin
                                                  : before + (unsigned)(h * w.tiles + t) * (w.steps + begin_of(tile)) + begin_of(tile);
                    const Parts in(prompt ? big_units : units, prompt ? big_groups_of(big_groups, big_units) : groups_of(groups, units), first,
                                   prompt ? big_w.before(t + 1) - big_w.before(t) - kBigBegin : w.steps);
                    const std::vector<int> &have = (prompt ? big_slots : slots)[at];
                    CHECK(in.count >= 1 && (int)have.size() == in.count);
                    for (int p = 0; p < in.count; p++) {
                        if (in.count == 1) CHECK(have[p] == -1);
                        else {
                            CHECK(have[p] == in.slot(p) && in.slot(p) >= 0 && in.slot(p) < 2 * (prompt ? big_groups : groups));
                            CHECK((prompt ? big_used : used)[in.slot(p)]++ == 0);
                        }
                    }
                }
            before += w.units;
            big_before += big_w.units(Hkv);
        }
    }
};

int main(int argc, char **argv)
{
    std::mt19937 r(atoi(argv[1]));
    auto draw = [&](int lo, int hi) { return lo + (int)(r() % (unsigned)(hi - lo + 1)); };
    for (int page = 16; page <= 256; page += 16)
        for (int x = 0; x < kEntries * page; x++) CHECK(page_of(x, magic_of(page)) == x / page);
    const int heads[] = {1, 1, 2, 3, 4, 7, 8, 16, 33, 40, 72, 130, 200};
    for (int round = 0; round < 120; round++) {
        Batch t;
        t.G = heads[draw(0, 12)], t.Hkv = draw(1, 5), t.page = 16 * draw(1, 16);
        const int kind = draw(0, 2), most = draw(1, draw(0, 1) ? 6 : kind ? 700 : 120);
        t.few = kind == 0 ? INT32_MAX : kind == 1 ? 32 : 0;
        t.groups = draw(1, 40) * draw(1, 20), t.big_groups = 8 * draw(1, 64);
        const int B = draw(1, draw(0, 3) ? 12 : 90);
        for (int b = 0; b < B; b++) t.seqs.push_back({draw(0, 3) ? draw(0, most) : most, draw(0, draw(0, 2) ? 2000 : 20)});
        t.check(kind == 0 && draw(0, 1) ? 16 : 32);
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("shares")
    (d / "t.cpp").write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined,address", "-fno-sanitize-recover", "-Wall", "-Werror", "-I" + CSRC,
                           str(d / "t.cpp"), "-o", str(d / "t")])
    return str(d / "t")


@pytest.mark.parametrize("seed", range(4))
def test_all_work_is_done_once_and_no_page_is_looked_up_that_is_not_there(program, seed):
    r = subprocess.run([program, str(seed)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
