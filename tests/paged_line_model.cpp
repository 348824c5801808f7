// Runs the paged attention's own share and page arithmetic (csrc/paged_line.h) over random and extreme lines and checks it against the plain
// statement of what it stands for. usage: paged_line_model few|tickets|tm|large|pages SEED
#include "paged_line.h"

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

using namespace flb;
typedef std::mt19937 Rng;
static uint32_t pick(Rng &g, uint32_t lo, uint32_t hi) { return lo + (uint32_t)(((uint64_t)g() << 32 | g()) % ((uint64_t)hi - lo + 1)); }
#define CHECK(x) do { if (!(x)) { std::printf("failed: %s (line %d)\n", #x, __LINE__); return 1; } } while (0)

// Runs of tiles on a line: every tile is one CTA's, no share is empty, a run's CTAs are first_of .. last_of, and a CTA that goes on with a run
// has it in front of its others (its record is the one of tiles that began before).
static int few(Rng &g) {
    for (int it = 0; it < 20000; ++it) {
        const uint32_t n_run = pick(g, 1, 40), longest = 1u << pick(g, 0, 9), ctas = pick(g, 1, 300), snap = it & 1 ? kSnap : 0;
        std::vector<uint32_t> begin(1, 0);
        for (uint32_t i = 0; i < n_run; ++i) begin.push_back(begin.back() + pick(g, 1, longest));
        const uint32_t units = begin.back();
        const Shares sh = few_shares(units, ctas);
        CHECK(sh.n >= 1 && sh.n <= ctas && sh.n <= units && share_lo(sh, sh.n) == units);
        std::vector<uint32_t> edge;
        for (uint32_t c = 0, run = 0; c <= sh.n; ++c) {
            uint32_t at = share_lo(sh, c);
            if (edge_moves(sh, c)) {
                while (begin[run + 1] <= at) ++run;
                at = snapped(sh, snap, at, begin[run], begin[run + 1]);
            }
            CHECK(c == 0 ? at == 0 : at > edge.back());
            edge.push_back(at);
        }
        CHECK(edge.back() == units);
        std::vector<uint32_t> begins(sh.n, 0);
        for (uint32_t r = 0; r < n_run; ++r) {
            const uint32_t b = begin[r], e = begin[r + 1];
            uint32_t first = ~0u, last = 0;
            for (uint32_t c = 0; c < sh.n; ++c)
                if (edge[c] < e && edge[c + 1] > b) {
                    if (first == ~0u) first = c;
                    last = c;
                }
            CHECK((sh.each < 2 ? owner_of(sh, b) : first_of(sh, snap, b, e)) == first);
            CHECK((sh.each < 2 ? owner_of(sh, e - 1) : last_of(sh, snap, b, e)) == last);
            CHECK(edge[first] <= b);
            for (uint32_t c = first + 1; c <= last; ++c) CHECK(edge[c] > b && edge[c] < e);
            if (last > first) CHECK(begins[first]++ == 0);   // (one run at most begins in a CTA and goes on: one ticket, one second record)
        }
    }
    return 0;
}
// Whoever arrives last, and whoever gave up: the ticket is zero again, one CTA is the last, and it adds records only where all are there.
static int tickets(Rng &g) {
    for (int it = 0; it < 20000; ++it) {
        const uint32_t pieces = pick(g, 1, 296), rare = pick(g, 1, 400);
        uint32_t ticket = 0, lasts = 0;
        bool any_gave_up = false, added = false;
        for (uint32_t i = 0; i < pieces; ++i) {
            const bool gave_up = pick(g, 1, rare) == 1;
            any_gave_up |= gave_up;
            const uint32_t before = ticket;
            ticket += ticket_step(gave_up);
            if (ticket_last(before, pieces)) {
                ++lasts;
                ticket = 0;
                added = ticket_complete(before, gave_up);
            }
        }
        CHECK(ticket == 0 && lasts == 1 && added == !any_gave_up);
    }
    return 0;
}
// Blocks of rows: every tile is one CTA's, and the CTAs between the owners of a block's first and last tile have at least one each.
static int tm(Rng &g) {
    for (int it = 0; it < 20000; ++it) {
        const uint32_t n_block = pick(g, 1, 60), longest = 1u << pick(g, 0, 8), ctas = pick(g, 1, 200), front = pick(g, 0, 12);
        std::vector<uint32_t> base(1, 0), tiles, per;
        for (uint32_t i = 0; i < n_block; ++i) {
            tiles.push_back(pick(g, 1, longest));
            per.push_back(pick(g, 1, 2));
            base.push_back(base.back() + front + tiles[i] * per[i]);
        }
        const Shares sh = tm_shares(base.back(), ctas);
        CHECK(base.back() < 2 || (sh.n >= 1 && share_lo(sh, sh.n) == base.back()));
        std::vector<bool> used(2 * sh.n, false);
        for (uint32_t i = 0; i < n_block && sh.n; ++i) {
            const uint32_t f = base[i] + front, c0 = owner_of(sh, f), c1 = owner_of(sh, f + (tiles[i] - 1) * per[i]);
            uint32_t next = 0;
            for (uint32_t c = 0; c < sh.n; ++c) {
                const uint32_t t0 = tile_at_unit(share_lo(sh, c), f, tiles[i], per[i]), t1 = tile_at_unit(share_lo(sh, c + 1), f, tiles[i], per[i]);
                CHECK((t0 < t1) == (c >= c0 && c <= c1));
                if (t0 < t1) { CHECK(t0 == next); next = t1; }
                // a CTA that goes on with a block has no tile of one in front of it
                if (t0 < t1 && t0) CHECK(share_lo(sh, c) > f);
            }
            CHECK(next == tiles[i]);
            // its records are each in a place of their own, where the CTA has it: the first of its pieces, or one behind
            for (uint32_t c = c0; c <= c1 && c1 > c0; ++c) {
                bool in_front = false;   // tiles of a block in front of this one
                for (uint32_t j = 0; j < i; ++j) {
                    const uint32_t fj = base[j] + front;
                    in_front |= tile_at_unit(share_lo(sh, c), fj, tiles[j], per[j]) < tile_at_unit(share_lo(sh, c + 1), fj, tiles[j], per[j]);
                }
                const uint32_t at = record_index(c0, c - c0, c == c0 && in_front);
                CHECK(at == 2 * c + in_front && (c == c0 || !in_front) && at < 2 * sh.n && !used[at]);
                used[at] = true;
            }
        }
    }
    return 0;
}
// Lines up to the last that 32 bits hold.
static int large(Rng &g) {
    for (int it = 0; it < 200000; ++it) {
        const uint32_t units = it & 1 ? 0xFFFFFFFFu - pick(g, 0, 3) : pick(g, 1u << 31, 0xFFFFFFFFu), ctas = pick(g, 1, 592);
        for (const Shares &sh : {few_shares(units, ctas), tm_shares(units, ctas), shares_of(units, ctas)}) {
            CHECK(sh.n && (uint64_t)sh.each * sh.n + sh.more == units && share_lo(sh, sh.n) == units);
            const uint32_t u = it & 2 ? units - 1 - pick(g, 0, 3) : pick(g, 0, units - 1), c = owner_of(sh, u);
            CHECK(c < sh.n && share_lo(sh, c) <= u && u < share_lo(sh, c + 1));
            CHECK(owner_of(sh, share_lo(sh, c)) == c && owner_of(sh, share_lo(sh, c + 1) - 1) == c);
        }
        const uint32_t front = units - 9;
        CHECK(tile_at_unit(units, front, 5, 2) == 5 && tile_at_unit(units, front, 100, 1) == 9 && tile_at_unit(front, front, 5, 2) == 0);
    }
    return 0;
}
// The group of rows that a copy reads lies inside the pool for pages inside it, whatever 32 bits a table holds, and no product passes 32 bits.
static int pages(Rng &g) {
    for (int it = 0; it < 200000; ++it) {
        const uint32_t shift = pick(g, 4, 8), n_kv = it & 1 ? pick(g, 1, 1024) : pick(g, 1, 16);
        const uint64_t most = ((1ull << 31) - 1) / ((uint64_t)n_kv << shift);   // (rows of a pool are below 2^31)
        const uint32_t n_pages = it & 2 ? (uint32_t)most : pick(g, 1, (uint32_t)most), behind = pool_groups(n_pages, n_kv, shift);
        CHECK(behind == (uint64_t)n_pages * n_kv * (1u << shift) / 8 && behind < 1u << 28);
        const int32_t tried[] = {0, (int32_t)(n_pages - 1), (int32_t)n_pages, 1 << 30, -1, INT32_MIN, INT32_MAX, (int32_t)g()};
        for (int32_t page : tried) {
            CHECK(page_there(page, n_pages) == (page >= 0 && (uint32_t)page < n_pages));
            if (!page_there(page, n_pages)) continue;
            const uint32_t hkv = pick(g, 0, n_kv - 1), key = g() & ~7u, at = page_group((uint32_t)page, n_kv, hkv, shift, key);
            CHECK(at < behind && (uint64_t)at * 8 == (((uint64_t)page * n_kv + hkv) << shift) + key % (1u << shift));
        }
    }
    return 0;
}

int main(int argc, char **argv) {
    if (argc != 3) return 2;
    Rng g((uint32_t)std::atoi(argv[2]));
    const char *w = argv[1];
    return !std::strcmp(w, "few") ? few(g) : !std::strcmp(w, "tickets") ? tickets(g) : !std::strcmp(w, "tm") ? tm(g) : !std::strcmp(w, "large") ? large(g) : !std::strcmp(w, "pages") ? pages(g) : 2;
}
