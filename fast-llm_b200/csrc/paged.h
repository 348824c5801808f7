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
    uint32_t n_seq, max_blocks, n_tokens, max_new, n_pages, page_shift;
    uint32_t n_kv, group, half;     // half: activations are f16
    uint32_t few_rows;              // sequences of at most so many rows over a KV head are the first kernel's, the others the second's
    float scale;
};

// Sequences of few rows over a KV head (mma.sync: attn_paged.cu) and of many (tcgen05: attn_paged_tm.cu). kmap and vmap are filled in there. us of
// both at 4 x 65000, 32 x 4000 and 1 x 8000 keys, 8 KV heads: 4 rows 150, 76, 15 and 212, 136, 34 (f16: 158, 92, 29); 16 rows 165, 92, 27 and
// 215, 137, 34 (f16: 158, 92, 29).
constexpr uint32_t kFewRows = 16;
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
