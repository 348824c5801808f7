// Paged attention: the whole-number arithmetic that decides which CTA works on what, where a page lies and when a block's records are complete.
// No CUDA in it, so that tests run the kernels' own functions on the CPU, over sizes that no call of a test reaches (tests/paged_line_model.cpp).
#pragma once
#include <cstdint>

#if defined(__CUDACC__)
#define FLB_HD __host__ __device__ __forceinline__
#else
#define FLB_HD inline
#endif

namespace flb {

FLB_HD uint32_t lesser(uint32_t a, uint32_t b) { return a < b ? a : b; }

// ---- shares: the line's units over the CTAs ----------------------------------------------------------------------------
// Equal shares up to one unit over n CTAs; none is empty (n <= units). 32 bits: a call with 2^32 units or more is refused.
struct Shares { uint32_t n, each, more; };   // the first `more` CTAs have one unit more than `each`
FLB_HD Shares shares_of(uint32_t units, uint32_t ctas) {
    const uint32_t n = lesser(ctas, units);
    return n ? Shares{n, units / n, units % n} : Shares{0, 0, 0};
}
FLB_HD uint32_t share_lo(const Shares &s, uint32_t c) { return s.each * c + lesser(c, s.more); }
FLB_HD uint32_t owner_of(const Shares &s, uint32_t u) {   // the CTA whose share holds unit u
    const uint32_t front = s.more * (s.each + 1);
    return u < front ? u / (s.each + 1) : s.more + (u - front) / s.each;
}

// ---- few rows (attn_paged.cu): a unit is a tile, the tiles b .. e - 1 of a sequence over one KV head a run ------------------
// An end of a share that lies in a run, within kSnap tiles of b or e, moves there: a CTA with a few
// tiles of another head builds rows of q, leaves a record, is the last to arrive at both and adds the records of both (one sequence over 8000
// keys 17.0 us, moved 15.1; 4 over 1023 13.0, 10.2; 8 over 2000 17.6, 15.4; 16 over 5500 to 8192, where shares are long, 78.1, 78.6). Up by
// less than half a share, down by half of one at most, so that none gets empty.
constexpr uint32_t kSnap = 4;
// The line over at most `ctas` CTAs: where shares are that small no more of them than keep the largest one, which leaves fewer records. (Longer
// shares: all of them, for the HBM's sake; 16 x 5500 to 8192 keys 78.5 us, 79.9 with 292 CTAs of 296.)
FLB_HD Shares few_shares(uint32_t units, uint32_t ctas) {
    const uint32_t most = units / ctas + (units % ctas ? 1u : 0u);
    return shares_of(units, most == 0 || most > 2 * kSnap ? ctas : units / most + (units % most ? 1u : 0u));
}
FLB_HD uint32_t snapped(const Shares &sh, uint32_t snap, uint32_t at, uint32_t b, uint32_t e) {
    const uint32_t down = at - b, up = e - at;
    const bool may_down = down <= snap && 2 * down <= sh.each, may_up = up <= snap && 2 * up < sh.each;
    return may_down && (!may_up || down <= up) ? b : may_up ? e : at;
}
// The end of CTA c's share in front, which lies in the run b .. e
FLB_HD bool edge_moves(const Shares &sh, uint32_t c) { return c != 0 && c != sh.n && sh.each >= 2; }   // (shares of a tile cannot move: the smallest calls, 9.8 -> 9.4 us)
// The first and the last CTA of a run, where shares are two tiles at least (else owner_of: ends do not move)
FLB_HD uint32_t first_of(const Shares &sh, uint32_t snap, uint32_t b, uint32_t e) {
    const uint32_t c = owner_of(sh, b), hi = share_lo(sh, c + 1);
    return hi < e && snapped(sh, snap, hi, b, e) == b ? c + 1 : c;
}
FLB_HD uint32_t last_of(const Shares &sh, uint32_t snap, uint32_t b, uint32_t e) {
    const uint32_t c = owner_of(sh, e - 1), lo = share_lo(sh, c);
    return lo > b && snapped(sh, snap, lo, b, e) == e ? c - 1 : c;
}

// A run's ticket, zero between launches: CTAs that arrived in the low half, those of them that gave up a wait, and left no record, in the
// high half. The last to arrive resets it, and adds the records where there are all of them.
FLB_HD uint32_t ticket_step(bool gave_up) { return gave_up ? 0x10001u : 1u; }
FLB_HD bool ticket_last(uint32_t before, uint32_t pieces) { return (before & 0xFFFFu) == pieces - 1; }
FLB_HD bool ticket_complete(uint32_t before, bool gave_up) { return before >> 16 == 0 && !gave_up; }

// ---- many rows (attn_paged_tm.cu): a block of rows is `front` units, then tile_units for every tile ----------------------------
// Two units at least, so that every CTA between a block's first and last one has a tile of it.
FLB_HD Shares tm_shares(uint32_t units, uint32_t ctas) { return shares_of(units, lesser(ctas, units / 2)); }
// A tile is the CTA's whose share holds its first unit: the first tile at or behind unit `at`, of a block whose tiles begin at unit `front`.
FLB_HD uint32_t tile_at_unit(uint32_t at, uint32_t front, uint32_t tiles, uint32_t tile_units) {
    return at > front ? lesser(tiles, (at - front + tile_units - 1) >> (tile_units - 1)) : 0u;   // (1 or 2)
}
// The record of a block's CTA `first + i` is its second (slot 1) where the block begins behind another one's tiles, which only the first
// CTA's can; every CTA notes which of its two it left: left[2 cta + slot].
FLB_HD uint32_t record_index(uint32_t first, uint32_t i, uint32_t slot) { return 2 * (first + i) + (i ? 0u : slot); }

// ---- pages ----------------------------------------------------------------------------------------------------------
// The pool in groups of 8 rows: where the group of row `row` of a page over KV head hkv lies. Pages outside the pool (and keys behind the last):
// behind its end, where copies bring zeros. The pool's rows are below 2^31.
FLB_HD uint32_t pool_groups(uint32_t n_pages, uint32_t n_kv, uint32_t page_shift) { return n_pages * n_kv * ((1u << page_shift) >> 3); }
FLB_HD uint32_t page_group(uint32_t page, uint32_t n_kv, uint32_t hkv, uint32_t page_shift, uint32_t row) {
    return (page * n_kv + hkv) * ((1u << page_shift) >> 3) + ((row & ((1u << page_shift) - 1u)) >> 3);
}
FLB_HD bool page_there(int32_t page, uint32_t n_pages) { return (uint32_t)page < n_pages; }

} // namespace flb
