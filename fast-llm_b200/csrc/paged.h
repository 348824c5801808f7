// Paged KV cache: launch interface between paged.cu (C ABI, plan, append) and the attention kernels over pages.
//
// Layout: K and V are pools of pages, each [n_pages][n_kv_head][page_size][head_dim] f16, so that a page of one KV head is one
// contiguous piece as in the unpaged cache. Slot p * page_size + r is row r of page p. A sequence's block table names its pages
// in order: key j lies in slot table[j / page_size] * page_size + j % page_size.
#pragma once
#include "../../include/fl_b200.h"
#include "kernels.h"
#include "paged_line.h"

namespace flb {

constexpr uint32_t kPagedMaxSeq = 4096;   // sequences of a call: the plan keeps three prefix sums of them in shared memory

// ---- attention over pages -------------------------------------------------------------------------------------------
// Rows: row r of a sequence with n new tokens is token r / group, query head hkv * group + r % group (group = n_q_head / n_kv_head).
// Token i of n attends keys 0 .. kv_len - n + i. A block of rows over one KV head walks tiles of keys; the tiles of all blocks lie
// on one line and every CTA takes an equal, contiguous piece of it, so that ragged batches load all SMs alike. A block that several
// CTAs share leaves one record per CTA; the CTA that arrives last, or the launch behind, adds them in order (no CTA waits for another).
// A block that several CTAs of attn_paged_tm.cu share, noted by the one that begins it.
struct PagedTmBlock {
    uint32_t records, slot, first, row0, rows, hkv;   // records: CTAs; 0: none. slot: of the first CTA's record
    int32_t past;
};
struct PagedAttnArgs {
    CUtensorMap kmap, vmap;         // tensor_map_groups_swz: one copy per page; the layout of ldmatrix and tcgen05 operands alike
    const void *q;
    void *out;
    float2 *lse;                    // optional
    const int32_t *table, *q_start, *kv_len;
    float *part, *part_tm;          // records
    PagedTmBlock *blocks;           // one per CTA, then two words each: its records that are complete
    uint32_t *tickets;              // zero between launches (attn_paged.cu)
    uint32_t *status;
    uint64_t q_stride, out_stride;  // elements between tokens
    uint32_t spare;                 // see few_limit; 0: no sequence can have many rows
    uint32_t n_seq, max_blocks, n_tokens, max_new, n_pages, page_shift;
    uint32_t n_kv, group, half;     // half: activations are f16
    float scale;
};

// Sequences of few rows over a KV head (mma.sync: attn_paged.cu) and of many (tcgen05: attn_paged_tm.cu). kmap and vmap are filled in
// there. 16 is what the first kernel's instances hold. us of both at 4 x 65000, 32 x 4000 and 1 x 8000 keys, 8 KV heads of 128, pages of
// 16: 4 rows 166, 91, 17 and 243, 197, 40 (f16 166, 89, 16 and 187, 143, 32); 16 rows 200, 150, 29 and 257, 181, 34 (f16 200, 126, 29 and
// 188, 134, 30).
constexpr uint32_t kFewRows = 16;
// Up to 32 sequences, of few rows and of many: the second kernel takes all of them where those of few rows are less work than a launch of
// their own in front of it, in tiles of 128 keys; a sequence's start and end over a KV head count as 60. us with two launches and with one,
// 8 KV heads of 128 dimensions, single tokens over so many keys: f32, beside 500 tokens over 4000 keys 8 x 4000 133 and 122, 12 x 4000 144
// and 138, 16 x 4000 151 and 149, 1 x 65000 161 and 143, 2 x 65000 196 and 202; beside 30 over 1000 12 x 2000 49 and 61; beside 200 over
// 500 28 x 300 40 and 65. f16, whose tiles take the second kernel half as long: 8 x 4000 100 and 85, 16 x 4000 118 and 107, 2 x 65000 162
// and 148, 12 x 2000 44 and 45, 28 x 300 37 and 45; f16 and heads of 64: 8 x 4000 74 and 72, 16 x 4000 87 and 96.
constexpr uint32_t kSpareStart = 60, kSpare = 6500, kSpareHalf128 = 12000;
// Where the table's width bounds that work by as much as this the first kernel is not launched (4 x 8 tokens over 4096 keys 39.6 us, 36
// without). The price: single tokens in a call that allows more, as a recorded one may, run on the second kernel (1 x 8000 keys 24 us, 31
// so; 4 x 1000 18, 24).
constexpr uint32_t kSpareNoLaunch = 4000, kSpareAll = 0xffffffffu;
cudaError_t paged_few_init(void);
size_t paged_few_part_bytes(int sms);
cudaError_t launch_paged_few(PagedAttnArgs a, const void *k, const void *v, uint32_t head_dim, int sms, cudaStream_t stream);
cudaError_t paged_tm_init(void);
size_t paged_tm_part_bytes(int sms);
cudaError_t launch_paged_tm(PagedAttnArgs a, const void *k, const void *v, uint32_t head_dim, int sms, cudaStream_t stream);
constexpr uint32_t kPagedTickets = 1024;   // at least twice the SMs

#if defined(__CUDACC__)
// One sequence of an attention call, checked: n = 0 where its lengths do not fit the call (reported by `report`).
struct PagedSeq { uint32_t first, n; int32_t past; };   // past = kv_len - n; may be negative (rows without a key)
__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnArgs &a, uint32_t s, bool &bad) {
    const int32_t b = a.q_start[s], e = a.q_start[s + 1], len = a.kv_len[s];
    const uint64_t room = (uint64_t)a.max_blocks << a.page_shift;
    bad = b < 0 || e < b || (uint32_t)e > a.n_tokens || (uint32_t)(e - b) > a.max_new || len < 0 || (uint64_t)len > room;
    return bad ? PagedSeq{0, 0, 0} : PagedSeq{(uint32_t)b, (uint32_t)(e - b), len - (e - b)};
}
// The rows that a sequence of the first kernel has at most (lane i holds sequence i, of up to 32): none where the second one has others to
// work on and takes those too.
__device__ __forceinline__ uint32_t few_limit(const PagedAttnArgs &a, const PagedSeq &q) {
    if (a.spare == 0 || a.spare == kSpareAll) return a.spare ? 0u : kFewRows;
    const uint32_t rows = q.n * a.group, tiles = ((uint32_t)max(0, q.past + (int32_t)q.n) + 127) / 128;
    const uint32_t cost = rows && rows <= kFewRows ? min(min(tiles + kSpareStart, 1u << 16) * a.n_kv, 1u << 24) : 0u;   // (32 of them below 2^32)
    const uint32_t all = __reduce_add_sync(0xffffffffu, cost);
    return __any_sync(0xffffffffu, rows > kFewRows) && all <= a.spare ? 0u : kFewRows;
}

// Values of +inf, -inf and NaN (class 0, 1, 2) among the keys that only part of the rows attend: per class and dimension the
// first such key. A row that attends keys 0 .. lim is affected by those <= lim.
__device__ __forceinline__ float unfinite_of(const uint32_t *u, uint32_t dims, uint32_t d, int32_t lim) {
    const int32_t p = (int32_t)u[d], n = (int32_t)u[dims + d], x = (int32_t)u[2 * dims + d];   // (0x7fffffff: none)
    if (x <= lim || (p <= lim && n <= lim)) return __int_as_float(0x7fffffff);
    return p <= lim ? INFINITY : n <= lim ? -INFINITY : 0.f;
}

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x to 2^-22 of its value, 0 for -inf
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
#endif

} // namespace flb
