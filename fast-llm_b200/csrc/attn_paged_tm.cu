// Attention over a paged cache, many rows per sequence and KV head (prompt chunks, drafts): blocks of up to 256 rows (token,
// query head of the group) against tiles of 128 keys on tcgen05, scores and contexts in tensor memory.
//
// The mathematics are attn_paged.cu's: an online softmax in f32. f32 activations: q and the probabilities are two f16 parts each, so
// that a pair of row and key costs 8 D tensor flops instead of 4 D, and nothing else is rounded below 32 bits (small probabilities: see kShift). f16
// activations (Parts = 1): q as it is, the probabilities as one f16 (half a step of 2^-11, as the result).
//
// Bound by the chain scores - softmax - context of each lane. A tile of 128 keys and 256 rows, head_dim 128: about 3900 cycles for f16
// activations, 7600 for f32 (ncu's cycles of 2048 tokens over 30000 keys and of 4096 tokens, a block's start and end counted as six tiles); the
// tensor pipe is busy for 2100 and 4200 of them (53 and 40 % of the launches), the exponentials and conversions for 55 % of the first. Measured
// (32/8 heads, device times): 2048 tokens over 30000 keys, f16, 990 us in a burst (1.05 PFLOP/s), 1160 under the power cap; 4096 tokens, f32, 343
// us (0.80 PFLOP/s of tensor work); 4 x 8 tokens over 4096 keys 35.6 us. Roles of a CTA (11 warps, one CTA per SM):
//   softmax (2 x 4 warps): "lane" l = its 128 rows, thread = row: scores out of tensor memory, maximum, exponentials, probabilities
//                          back over the scores' columns; at the end of a piece the contexts out
//   copy    (1 warp)     : K and V tiles into a ring of slots, one TMA box per page (attn_paged.cu)
//   tensor  (1 warp)     : scores S = Q K^T (Q, K in shared memory), context O += P V (P in tensor memory)
//   values  (1 warp)     : V tiles that hold keys which only part of the rows attend: keys behind the last are cleared, values that
//                          are not finite are taken out and noted (0 x NaN; see unfinite_of)
// While one lane's softmax runs the tensor cores work for the other: a block of more than 128 rows gives each lane 128 of them over the same
// tiles; a smaller block gives both lanes its rows, every other tile each, and their results are added in tensor memory.
// Tiles of all blocks lie on one line (sequence, KV head, block, tile) and every CTA takes an equal piece of it; the records of a block that
// several CTAs share are added by a launch of its own behind.
//
// The tensor cores truncate their running sum, 3.1e-8 of it per instruction in the mean; with f32 activations half of O's columns are therefore
// brought out at every tile, in turn, added in f32 to a buffer of the CTA's own that stays in L2, and start from zero: no sum in
// tensor memory is longer than three tiles (48 instructions). (us with a quarter at every tile, sums of up to eight: 4 x 8 tokens over 4096
// keys 32.7, now 35.2; 4096 tokens 310, 320; 1000 over 20000 keys 554, 603.) f16 activations: at every 128th tile, so that no sum is longer
// than 129 (1032 instructions, which cut off 2^-13 at most; uncut, rows of a million keys came out 0.7 % too small).
#include "common.cuh"
#include "paged.h"

#include <algorithm>

namespace flb {

namespace {

constexpr uint32_t kRowsL = 128, kTile = 128;
constexpr uint32_t kCopyWarp = 8, kTensorWarp = 9, kValueWarp = 10, kThreads = 11 * 32;
// Probabilities are 2^(x - ref), ref = maximum - 12 when it is set and kept while they stay below 2^15, which f16 holds. f16 has steps of 2^-24 at
// its lower end: a probability below 2^-14 of the row's largest is held to 2^-36 of that (half a step for each part), one below 2^-37 is lost.
constexpr float kShift = 12.f, kLag = 3.f;
constexpr uint32_t kOCol = 256, kTmemCols = 512;

template <int D, int Parts> struct Tm {
    static constexpr uint32_t kPart = kRowsL * D * 2;               // one part of a lane's q; a K or V tile
    static constexpr uint32_t kQ = 2 * Parts * kPart;
    static constexpr uint32_t kSlots = D == 64 ? 8 : Parts == 2 ? 3 : 5;
    static constexpr uint32_t kHead = 2048;                         // barriers and the like, in front
    static constexpr uint32_t kBytes = kHead + kQ + kSlots * kPart;
    static constexpr uint32_t kRecord = kRowsL * (D + 3);           // floats: [D / 4][128 rows][4], then references, sums, maxima
};
// A piece as the softmax warps use it, in shared memory (as registers its fields would cost a row of scores theirs).
struct Job {
    uint32_t valid, sm, n, t0;          // sm: small block; tiles t0 .. t0 + n - 1
    uint32_t first, row0, rows, hkv;    // the sequence's first token; the block's rows row0 .. row0 + rows - 1
    uint32_t whole, slot;               // the block is this CTA's alone; its record's
    int32_t past;
};
struct Walk { uint32_t pos, hi, few; };   // the share's units behind the piece; see few_limit
struct Block { uint32_t rows, tiles, units; int32_t keys; };
struct Piece {
    PagedSeq q;
    uint32_t seq, hkv, blk, n_blk;
    Block b;
    uint32_t t0, t1;
    uint32_t base;       // first unit of its block
};
struct Head {
    uint64_t full[8], empty[8], v_ready[8], s_full[2], p_full[2][2], o_done[2], q_full, drain;
    uint32_t start_seq, start_off, tmem, abort_flag, any_unfinite;
    Job job;
    Walk walk;
    Piece piece;
    union { uint32_t unfinite[3 * 128]; uint64_t sum[kThreads / 32]; };   // (the sums while the share is found)
};
static_assert(sizeof(Head) <= 2048, "head");

__device__ __forceinline__ bool try_bar(uint64_t *bar, uint32_t parity) { return mbar_try_wait(bar, parity); }
// A warp's wait: at most a second, and no longer once another role has given up.
__device__ __forceinline__ bool wait_slow(uint64_t *bar, uint32_t parity, uint32_t *status, volatile uint32_t *abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
        for (int i = 0; i < 4; ++i)
            if (__all_sync(0xffffffffu, try_bar(bar, parity))) return true;
        const bool late = globaltimer_ns() - t0 > kDefaultWaitNs, stop = *abort_flag != 0;
        if (__any_sync(0xffffffffu, late || stop)) {
            if (!stop) { atomicCAS(status, ST_OK, ST_WAIT_TIMEOUT); *abort_flag = 1u; }
            return false;
        }
    }
}
__device__ __forceinline__ void arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// 32 columns of the thread's lane of tensor memory; used after wait_ld
__device__ __forceinline__ void load32(uint32_t addr, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]),
          "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]),
          "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void load16(uint32_t addr, float *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]),
                   "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
                 : "r"(addr)
                 : "memory");
}
template <int N> __device__ __forceinline__ void wait_ld(float (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(r[i]));
}
__device__ __forceinline__ void store16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15])
                 : "memory");
}
// Shared-memory matrix descriptors, 128-byte swizzle. K-major: 8-row groups `sbo` bytes apart. MN-major: 64-element blocks `lbo` bytes
// apart, groups of 8 k `sbo` bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
                 "r"(accumulate)
                 : "memory");
}
// f32 result, f16 operands, M 128
__device__ __forceinline__ constexpr uint32_t idesc_of(uint32_t n, bool b_mn_major) { return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | (8u << 24); }

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// two f32 at once
struct F2 { uint64_t v; };
__device__ __forceinline__ F2 pair(float a, float b) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpair(F2 x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ F2 add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }

__device__ __forceinline__ void cut_at(float (&s)[32], int32_t valid) {   // columns behind `valid` are masked
#pragma unroll
    for (int c = 0; c < 32; ++c) s[c] = c <= valid ? s[c] : -INFINITY;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_of(const float (&s)[32]) {
    float t[4] = {max3(s[0], s[1], s[2]), max3(s[3], s[4], s[5]), max3(s[6], s[7], s[8]), max3(s[9], s[10], s[11])};
#pragma unroll
    for (int c = 12; c < 28; c += 8)
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = max3(t[j], s[c + 2 * j], s[c + 2 * j + 1]);
    return max3(max3(t[0], s[28], s[29]), max3(t[1], s[30], s[31]), fmaxf(t[2], t[3]));
}
__device__ __forceinline__ void add4(float4 *at, const float4 &v) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
// A row's sums in memory (columns 32 c .. for the bits c of `out`) from one reference to another, which is returned.
__device__ __noinline__ float move_sums(float4 *mem, uint32_t out, float from, float to) {
    __threadfence();
    const float by = from == -INFINITY ? 0.f : exp2_fast(from - to);
    for (uint32_t c = 0; c < 32; ++c)
        if (out >> (c / 8) & 1u) {
            float4 *at = mem + c * kRowsL;
            const float4 v = __ldcg(at);
            __stcg(at, make_float4(v.x * by, v.y * by, v.z * by, v.w * by));
        }
    __threadfence();
    return to;
}
// 32 columns of the row's contexts out of tensor memory, where they start from zero, to their sum in memory, times `by`.
__device__ __forceinline__ void add_out(uint32_t to, float4 *mem, uint32_t c4, float by, bool adds) {
    float o[32];
    load32(to + 32 * c4, o);
    wait_ld(o);
    const uint32_t zero[16] = {};
    store16(to + 32 * c4, zero);
    store16(to + 32 * c4 + 16, zero);
    float4 *at = mem + 8 * c4 * kRowsL;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 v = make_float4(o[4 * j] * by, o[4 * j + 1] * by, o[4 * j + 2] * by, o[4 * j + 3] * by);
        if (adds) add4(at + j * kRowsL, v);
        else __stcg(at + j * kRowsL, v);
    }
}
__device__ __forceinline__ void scale_o(uint32_t at, uint32_t columns, float by) {
#pragma unroll 1
    for (uint32_t c = 0; c < columns; c += 32) {
        float o[32];
        load32(at + c, o);
        wait_ld(o);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(o[16 * h + j] * by);
            store16(at + c + 16 * h, w);
        }
    }
}
// f16 activations: a half of the contexts goes out at steps n kOutHalf and n kOutHalf + 1, and comes back at the piece's end. What went out
// follows from the step, and the reference of the sums lies beside them, so that the loop over the tiles holds nothing of it. (us at 4096
// tokens with heads of 64, and at 2048 tokens over 30000 keys: without 152, 970; this 157, 990; as a call of its own in the loop, every
// 64th tile, 167, 1010.)
constexpr uint32_t kOutHalf = 128;
__device__ __forceinline__ bool half_goes(uint32_t step) { return step >= kOutHalf && step % kOutHalf < 2; }
template <int D> __device__ __forceinline__ uint32_t halves_out(uint32_t steps) {   // in front of step `steps`: bit c: columns 32 c ..
    constexpr uint32_t kHalf = (1u << D / 64) - 1u;
    return (steps > kOutHalf ? kHalf : 0u) | (steps > kOutHalf + 1 ? kHalf << D / 64 : 0u);
}
template <int D> __device__ __forceinline__ float *half_sums(const PagedAttnArgs &a) {   // of the warp's lane: [D / 4][128 rows][4], a row each, references
    return a.part_tm + ((uint64_t)gridDim.x * 4 + blockIdx.x * 2 + (threadIdx.x >> 7)) * Tm<D, 1>::kRecord;
}
// The row's contexts times `by`, where that changes its reference to ref. (Out of line, as load_q and finish are: what they need in
// registers stays out of the loop over the tiles.)
template <int D, int Parts> __device__ __noinline__ void change_o(const PagedAttnArgs &a, uint32_t to, float by, uint32_t step, float ref) {
    if (__any_sync(0xffffffffu, by != 1.f)) scale_o(to, D, by);
    if (Parts == 2 || !half_goes(step)) return;
    wait_st();
    const uint32_t out = halves_out<D>(step), r = threadIdx.x & (kRowsL - 1);
    float *sums = half_sums<D>(a), *at = sums + (D + 1) * kRowsL + r;
    float4 *mem = reinterpret_cast<float4 *>(sums) + r;
    if (out) {
        const float from = __ldcg(at);
        if (from != ref) move_sums(mem, out, from, ref);
    }
    __stcg(at, ref);
#pragma unroll 1
    for (uint32_t c4 = (step & 1u) * (D / 64); c4 < ((step & 1u) + 1) * (D / 64); ++c4) add_out(to, mem, c4, 1.f, out >> c4 & 1u);
}
template <int D> __device__ __noinline__ void halves_back(const PagedAttnArgs &a, uint32_t to, uint32_t steps, float ref) {
    const uint32_t out = halves_out<D>(steps), r = threadIdx.x & (kRowsL - 1);
    const float *sums = half_sums<D>(a);
    __threadfence();   // (the additions come before the loads)
    const float from = __ldcg(sums + (D + 1) * kRowsL + r), by = from == ref ? 1.f : exp2_fast(from - ref);
#pragma unroll 1
    for (uint32_t c = 0; c < D / 32; ++c)
        if (out >> c & 1u) {
            float4 v[8];
            float o[32];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __ldcg(reinterpret_cast<const float4 *>(sums) + (8 * c + j) * kRowsL + r);
            load32(to + 32 * c, o);
            wait_ld(o);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[16];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 x = v[4 * h + j];
                    const float *y = o + 16 * h + 4 * j;
                    w[4 * j] = __float_as_uint(fmaf(x.x, by, y[0]));
                    w[4 * j + 1] = __float_as_uint(fmaf(x.y, by, y[1]));
                    w[4 * j + 2] = __float_as_uint(fmaf(x.z, by, y[2]));
                    w[4 * j + 3] = __float_as_uint(fmaf(x.w, by, y[3]));
                }
                store16(to + 32 * c + 16 * h, w);
            }
        }
    wait_st();
}
// 32 scores to probabilities, in place in tensor memory (at): 2^(s f + m) as f16, hi parts in the first 16 columns and, with two parts,
// lo parts in the others; sum += them. The hi part is the value cut off after 10 bits of mantissa, so that
// the lo part needs no conversion back: both together keep 21 bits (of small ones fewer: see kShift).
template <int Parts> __device__ __forceinline__ void exp_chunk(const float (&s)[32], F2 f, F2 m, F2 (&sum)[2], uint32_t at) {
    uint32_t ph[16], pl[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        float y0, y1;
        unpair(fma2(pair(s[2 * j], s[2 * j + 1]), f, m), y0, y1);
        const float e0 = exp2_fast(y0), e1 = exp2_fast(y1);
        sum[j & 1] = add2(sum[j & 1], pair(e0, e1));
        if (Parts == 2) {
            const float h0 = __uint_as_float(__float_as_uint(e0) & 0xFFFFE000u), h1 = __uint_as_float(__float_as_uint(e1) & 0xFFFFE000u);
            float l0, l1;
            unpair(fma2(pair(h0, h1), pair(-1.f, -1.f), pair(e0, e1)), l0, l1);
            ph[j] = half2_bits(h0, h1);
            pl[j] = half2_bits(l0, l1);
        } else {
            ph[j] = half2_bits(e0, e1);
        }
    }
    store16(at, ph);
    if (Parts == 2) store16(at + 16, pl);
}

// 32 rows (16, half) from global memory, as f16 parts into shared memory (K-major, 128-byte swizzle), every row times a power of two that
// brings its largest value to [2^11, 2^12): 8 lanes a row, rows i, i + 4, i + 8, i + 12 at a time, whose lines lie in both halves of the
// banks. A warp; lane t has row row0 + t: src is where that begins; returns what its scores are to be multiplied by (exponents of 2).
template <int D, int Parts>
__device__ __noinline__ float load_q(const PagedAttnArgs &a, uint8_t *dst, uint64_t src, uint32_t row0, uint32_t rows, bool half) {
    constexpr int V = 4, K = D / 32, kBatch = 4;   // values of a load, loads of a lane and row, groups of 4 rows in flight
    const uint32_t lane = threadIdx.x & 31u, sub = lane & 7u, group = lane >> 3;
    auto row_of = [&](uint32_t i) { return (i & 3u) + 4 * group + 16 * (i >> 2); };
    float f = 0.f;
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < (half ? 4u : 8u); i0 += kBatch) {
        float x[kBatch][K][V];
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
            const uint32_t rr = row_of(i0 + i);
            const uint64_t at = __shfl_sync(0xffffffffu, src, rr);
            const bool there = row0 + rr < rows;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const uint32_t d = (8 * k + sub) * V;
                if (Parts == 1) {
                    const uint2 y = there ? __ldg(reinterpret_cast<const uint2 *>((const __half *)a.q + at + d)) : make_uint2(0u, 0u);
                    const float2 y0 = __half22float2(*reinterpret_cast<const __half2 *>(&y.x)), y1 = __half22float2(*reinterpret_cast<const __half2 *>(&y.y));
                    x[i][k][0] = y0.x; x[i][k][1] = y0.y; x[i][k][2] = y1.x; x[i][k][3] = y1.y;
                } else {
                    const float4 y = there ? __ldg(reinterpret_cast<const float4 *>((const float *)a.q + at + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[i][k][0] = y.x; x[i][k][1] = y.y; x[i][k][2] = y.z; x[i][k][3] = y.w;
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
            const uint32_t rr = row0 + row_of(i0 + i);
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) top = fmaxf(top, fabsf(x[i][k][j]));
#pragma unroll
            for (int o = 4; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = min(126, max(-116, 138 - (int)(__float_as_uint(top) >> 23)));   // (-116: the largest f32; 2^-126 is a normal one)
            const float up = __uint_as_float((uint32_t)(e + 127) << 23);
            const float mine = fmaxf(a.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - e) << 23), 1e-37f);
            const float got = __shfl_sync(0xffffffffu, mine, (lane >> 2 & 3u) * 8);
            if ((lane & 3u) + 4 * (lane >> 4) == i0 + i) f = got;
            {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const uint32_t d = (8 * k + sub) * V;
                    uint8_t *to = dst + (d >> 6) * (kRowsL * 128) + (rr >> 3) * 1024 + (rr & 7u) * 128 + (((((d & 63u) >> 3) ^ rr) & 7u) << 4) + (d & 7u) * 2;
                    const float u0 = x[i][k][0] * up, u1 = x[i][k][1] * up, u2 = x[i][k][2] * up, u3 = x[i][k][3] * up;
                    const __half2 h0 = __floats2half2_rn(u0, u1), h1 = __floats2half2_rn(u2, u3);
                    *reinterpret_cast<uint2 *>(to) = make_uint2(*reinterpret_cast<const uint32_t *>(&h0), *reinterpret_cast<const uint32_t *>(&h1));
                    if (Parts == 2) {
                        const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
                        *reinterpret_cast<uint2 *>(to + Tm<D, Parts>::kPart) = make_uint2(half2_bits(u0 - b0.x, u1 - b0.y), half2_bits(u2 - b1.x, u3 - b1.y));
                    }
                }
            }
        }
    }
    return f;
}

// Rows of results through shared memory, so that a warp stores whole rows: 16-byte pieces of row r at (piece ^ r).
template <int D, int Parts> __device__ __forceinline__ void stage_put(uint8_t *stage, uint32_t r, uint32_t c, const float4 &v) {   // values 4 c ..
    if (Parts == 2) *reinterpret_cast<float4 *>(stage + r * (D * 4) + ((c ^ (r & (D / 4 - 1))) << 4)) = v;
    else *reinterpret_cast<uint2 *>(stage + r * (D * 2) + (((c >> 1) ^ (r & (D / 8 - 1))) << 4) + (c & 1u) * 8) = make_uint2(half2_bits(v.x, v.y), half2_bits(v.z, v.w));
}
template <int D, int Parts> __device__ __forceinline__ void stage_out(const uint8_t *stage, void *out, uint32_t row0, uint32_t rows, uint64_t dst) {   // a warp's 32 rows
    constexpr uint32_t kRowBytes = D * 2 * Parts, kLanes = kRowBytes / 16;   // lanes of a row
    const uint32_t lane = threadIdx.x & 31u, c = lane % kLanes;
    __syncwarp();
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < 32; i0 += 8 * (32 / kLanes)) {
        uint4 v[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t r = row0 + i0 + j * (32 / kLanes) + lane / kLanes;
            v[j] = *reinterpret_cast<const uint4 *>(stage + r * kRowBytes + ((c ^ (r & (kLanes - 1))) << 4));
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t i = i0 + j * (32 / kLanes) + lane / kLanes;
            const uint64_t at = __shfl_sync(0xffffffffu, dst, i);
            if (row0 + i < rows) *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(out) + at * (2 * Parts) + c * 16) = v[j];
        }
    }
    __syncwarp();
}

// (max score, sum of exp(score - max)) of a row from its largest exponent - kShift and the sum relative to 2^from
__device__ __forceinline__ float2 lse_of(float highest, float from, float sum) {
    return highest == -INFINITY ? make_float2(highest, sum) : make_float2((highest + kShift) * 0.693147180559945309f, sum * exp2_fast(from - highest - kShift));
}

// ---- blocks, shares, pieces --------------------------------------------------------------------------------------------
// A block's length on the line: its tiles, those of a small block half as long as the others (both lanes work on different ones), and in
// front of them what its start and end cost in tiles (q in, contexts out). A tile is the CTA's whose share holds its first unit. (Tiles
// alone: a prompt of 4096 tokens, whose first blocks have a tile or two, 482 us.)
constexpr uint32_t kStart = 12;
__device__ __forceinline__ uint32_t tile_units(uint32_t rows) { return rows <= kRowsL ? 1u : 2u; }
__device__ __forceinline__ Block block_of(const PagedAttnArgs &a, const PagedSeq &q, uint32_t blk) {
    Block b;
    b.rows = min(2 * kRowsL, q.n * a.group - blk * 2 * kRowsL);
    b.keys = max(0, q.past + (int32_t)((blk * 2 * kRowsL + b.rows - 1) / a.group) + 1);
    b.tiles = max(1u, ((uint32_t)b.keys + kTile - 1) / kTile);
    b.units = kStart + b.tiles * tile_units(b.rows);
    return b;
}
__device__ __forceinline__ uint32_t blocks_of(const PagedAttnArgs &a, uint32_t few, const PagedSeq &q) {   // of this kernel: sequences of more than `few` rows
    const uint32_t rows = q.n * a.group;
    return rows > few ? (rows + 2 * kRowsL - 1) / (2 * kRowsL) : 0u;
}
// Tiles of every lane's sequence over one KV head; long ones are summed by the whole warp.
__device__ __forceinline__ uint64_t head_units(const PagedAttnArgs &a, uint32_t few, const PagedSeq &q, uint32_t lane) {
    const uint32_t n = blocks_of(a, few, q);
    uint64_t u = 0;
    if (n <= 4)
        for (uint32_t b = 0; b < n; ++b) u += block_of(a, q, b).units;
    for (uint32_t todo = __ballot_sync(0xffffffffu, n > 4); todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        PagedSeq x;
        x.first = 0;
        x.n = __shfl_sync(0xffffffffu, q.n, src);
        x.past = __shfl_sync(0xffffffffu, q.past, src);
        const uint32_t nb = __shfl_sync(0xffffffffu, n, src);
        uint64_t v = 0;
        for (uint32_t b = lane; b < nb; b += 32) v += block_of(a, x, b).units;
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == (uint32_t)src) u = v;
    }
    return u;
}

// The tiles of the piece that begins at w.pos, in the block in p; false: there are none.
__device__ __forceinline__ bool cut_piece(Walk &w, Piece &p) {
    const uint32_t front = p.base + kStart, per = tile_units(p.b.rows);
    p.t0 = tile_at_unit(w.pos, front, p.b.tiles, per);
    p.t1 = tile_at_unit(w.hi, front, p.b.tiles, per);
    w.pos = min(w.hi, p.base + p.b.units);
    return p.t0 < p.t1;
}
// The CTAs that the piece's block's tiles begin and end in.
__device__ __forceinline__ uint32_t owner_of_tile(const Shares &sh, const Piece &p, uint32_t tile) { return owner_of(sh, p.base + kStart + tile * tile_units(p.b.rows)); }
// The share's first block (a warp): p has its sequence, whose first unit is p.base. The KV head, then the block, 32 at a time. Whether
// the share has tiles of it.
__device__ __forceinline__ bool first_piece(const PagedAttnArgs &a, Walk &w, Piece &p) {
    const uint32_t lane = threadIdx.x & 31u;
    p.n_blk = blocks_of(a, w.few, p.q);
    uint32_t per_head = 0;
    for (uint32_t b = lane; b < p.n_blk; b += 32) per_head += block_of(a, p.q, b).units;
    per_head = __reduce_add_sync(0xffffffffu, per_head);
    p.hkv = (w.pos - p.base) / per_head;
    p.base += p.hkv * per_head;
    for (uint32_t b0 = 0;; b0 += 32) {
        const uint32_t t = b0 + lane < p.n_blk ? block_of(a, p.q, b0 + lane).units : 0u;
        uint32_t x = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, p.base + x > w.pos);
        if (behind) {
            const int at = __ffs(behind) - 1;
            p.blk = b0 + at;
            p.base += __shfl_sync(0xffffffffu, x - t, at);
            break;
        }
        p.base += __shfl_sync(0xffffffffu, x, 31);
    }
    p.b = block_of(a, p.q, p.blk);
    return cut_piece(w, p);
}
// The piece behind p.
__device__ __forceinline__ bool next_piece(const PagedAttnArgs &a, Walk &w, Piece &p) {
    do {
        if (w.pos >= w.hi) return false;
        p.base += p.b.units;
        if (++p.blk == p.n_blk) {
            p.blk = 0;
            if (++p.hkv == a.n_kv) {
                bool bad;
                p.hkv = 0;
                do { p.q = paged_seq(a, ++p.seq, bad); } while ((p.n_blk = blocks_of(a, w.few, p.q)) == 0);
            }
        }
        p.b = block_of(a, p.q, p.blk);
    } while (!cut_piece(w, p));
    return true;
}
// A small block: both lanes have its rows, lane l the tiles t0 + l, t0 + l + 2, ..
__device__ __forceinline__ bool small(const Piece &p) { return p.b.rows <= kRowsL; }
// The order of a piece's copies is that in which the tensor warp first needs them: K0 V0 K1 V1 .. (both lanes on one tile),
// K0 K1 V0 K2 V1 K3 .. (every other tile each); n tiles.
__device__ __forceinline__ uint32_t k_index(bool sm, uint32_t t) { return sm ? (t ? 2 * t - 1 : 0) : 2 * t; }
__device__ __forceinline__ uint32_t v_index(bool sm, uint32_t t, uint32_t n) { return sm ? min(2 * t + 2, 2 * n - 1) : 2 * t + 1; }
__device__ __forceinline__ uint32_t copy_at(bool sm, uint32_t i, uint32_t n, bool &v) {   // the tile of copy i
    v = sm ? i == 2 * n - 1 || (i && !(i & 1u)) : i & 1u;
    return !sm ? i >> 1 : i == 2 * n - 1 ? n - 1 : v ? (i - 2) / 2 : (i + 1) / 2;
}
// Whether a tile holds keys that not all rows of the block attend.
__device__ __forceinline__ bool partly(const PagedAttnArgs &a, const Piece &p, uint32_t tile) {
    return (int32_t)((tile + 1) * kTile) > p.q.past + (int32_t)(p.blk * 2 * kRowsL / a.group) + 1;
}

__device__ __forceinline__ void bar_both() { asm volatile("bar.sync 1, 256;" ::: "memory"); }   // the softmax warps
// The same, and whether any of their threads says yes: what all of them then go by, whatever another role still writes.
__device__ __forceinline__ bool bar_both_any(bool yes) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((uint32_t)yes) : "memory");
    return r != 0;
}
__device__ __forceinline__ bool given_up(const Head &hd) { return *static_cast<const volatile uint32_t *>(&hd.abort_flag) != 0; }

// The rows of q of a piece to L2 (a warp).
template <int D, int Parts>
__device__ __noinline__ void prefetch_q(const PagedAttnArgs &a, const Piece p) {
    for (uint32_t i = threadIdx.x & 31u; i < p.b.rows; i += 32) {
        const uint32_t at = p.blk * 2 * kRowsL + i, tok = at / a.group, head = p.hkv * a.group + at - tok * a.group;
        const uint8_t *from = static_cast<const uint8_t *>(a.q) + ((p.q.first + tok) * a.q_stride + (uint64_t)head * D) * (2 * Parts);
        for (uint32_t c = 0; c < D * 2 * Parts; c += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(from + c));
    }
}
__device__ __forceinline__ uint32_t *records_left(const PagedAttnArgs &a) { return reinterpret_cast<uint32_t *>(a.blocks + gridDim.x); }
struct Sums { float ref, sum, highest, acc_ref; uint32_t out_of; };   // of a row
// The results of a lane's piece: the rows themselves, or a record. done: the lane has any, and they are in tensor memory.
template <int D, int Parts>
__device__ __noinline__ void finish(const PagedAttnArgs &a, Head &hd, uint8_t *q_s, const Sums s, bool done, uint32_t tmem) {
    using T = Tm<D, Parts>;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, l = warp >> 2, w4 = warp & 3u, r = tid & 127u;
    const uint32_t ts = tmem + (w4 * 32u << 16) + l * kTile, to = tmem + (w4 * 32u << 16) + kOCol + l * 128;
    const float4 *acc_mem = reinterpret_cast<const float4 *>(a.part_tm + ((uint64_t)gridDim.x * 4 + blockIdx.x * 2 + l) * T::kRecord) + r;
    const Job &job = hd.job;
    const bool sm = job.sm;
    const uint32_t row0 = job.row0 + (sm ? 0 : l * kRowsL), rows = min(kRowsL, sm ? job.rows : job.rows - min(job.rows, l * kRowsL));
    const uint32_t tok = (row0 + r) / a.group, head = job.hkv * a.group + (row0 + r) - tok * a.group;
    const bool there = r < rows, active = w4 * 32 < rows;
    const int32_t lim = there ? job.past + (int32_t)tok : 0x7fffffff;
    float ref = s.ref, sum = s.sum, highest = s.highest;
    // A small block: the second lane hands its sums to the first, in tensor memory, where its scores were
    float ref2 = -INFINITY, sum2 = 0.f, acc2_ref = -INFINITY;
    uint32_t out2 = 0;
    if (sm) {
        if (l && active) {
            const uint32_t w[16] = {__float_as_uint(ref), __float_as_uint(sum), __float_as_uint(highest), s.out_of, __float_as_uint(s.acc_ref)};
            store16(ts, w);
            wait_st();
        }
        fence_before();
        bar_both();
        fence_after();
        if (!l && active && job.n > 1) {
            float w[32];
            load32(ts + kTile, w);
            wait_ld(w);
            ref2 = w[0]; sum2 = w[1]; highest = fmaxf(highest, w[2]); out2 = __float_as_uint(w[3]); acc2_ref = w[4];
        }
    }
    if (done && active && !(sm && (l || given_up(hd)))) {   // (what the second lane hands over is its own where nobody gave up)
        const bool whole = job.whole, two = sm && job.n > 1;
        const float both = fmaxf(ref, ref2), w1 = ref == -INFINITY ? 0.f : exp2_fast(ref - both), w2 = ref2 == -INFINITY ? 0.f : exp2_fast(ref2 - both);
        const float all = fmaf(sum, w1, sum2 * w2), inv = lim < 0 ? 0.f : 1.f / all;
        float *rec = a.part_tm + (uint64_t)((blockIdx.x * 2 + job.slot) * 2 + l) * T::kRecord;
        // Rows go out through shared memory, where the lane's q was (a small block's lanes share the first q; the second is free).
        uint8_t *stage = q_s + (sm ? 1 : l) * Parts * T::kPart;
        const bool any_unfinite = hd.any_unfinite != 0;
        // 16 columns at a time (32 spill, and local memory is L2 here)
        struct Part { uint32_t at; const float4 *mem; uint32_t out; float keep; };
        const Part part1{to, acc_mem, s.out_of, s.acc_ref == ref ? 1.f : exp2_fast(s.acc_ref - ref)};
        const Part part2{to + 128, acc_mem + T::kRecord / 4, out2, acc2_ref == ref2 ? 1.f : exp2_fast(acc2_ref - ref2)};
        // (the sums in memory of the next columns are on their way meanwhile: 4 x 8 tokens over 4096 keys 37.3 us, 35.7 so)
        auto fetch = [&](const Part &p, int c, float4 (&x)[4]) {
            const bool acc = Parts == 2 && c < D / 16 && (p.out >> (c / 2) & 1u);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = acc ? __ldcg(p.mem + (4 * c + j) * kRowsL) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        auto add_part = [&](const Part &p, int c, float w, const float4 (&old)[4], float (&v)[16]) {   // v += w times the contexts of columns 16 c ..
            float o[16];
            load16(p.at + 16 * c, o);
            wait_ld(o);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = fmaf(o[j], w, v[j]);
            if (Parts == 2 && (p.out >> (c / 2) & 1u)) {
                const float keep = w * p.keep;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[4 * j] = fmaf(old[j].x, keep, v[4 * j]); v[4 * j + 1] = fmaf(old[j].y, keep, v[4 * j + 1]);
                    v[4 * j + 2] = fmaf(old[j].z, keep, v[4 * j + 2]); v[4 * j + 3] = fmaf(old[j].w, keep, v[4 * j + 3]);
                }
            }
        };
        float4 next1[4], next2[4];
        fetch(part1, 0, next1);
        fetch(part2, 0, next2);   // (nothing where there is no second part)
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
            float v[16] = {};
            float4 old1[4], old2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { old1[j] = next1[j]; old2[j] = next2[j]; }
            fetch(part1, c + 1, next1);
            fetch(part2, c + 1, next2);
            add_part(part1, c, two ? w1 : 1.f, old1, v);
            if (two) add_part(part2, c, w2, old2, v);
            if (any_unfinite)
#pragma unroll 1
                for (int j = 0; j < 16; ++j) {
                    const float u = unfinite_of(hd.unfinite, D, 16 * c + j, lim);
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] += i == j ? u : 0.f;
                }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!whole) __stcg(reinterpret_cast<float4 *>(rec) + (4 * c + j) * kRowsL + r, make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
                else stage_put<D, Parts>(stage, r, 4 * c + j, make_float4(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv));
            }
        }
        const float from = two ? both : ref, total_sum = two ? all : sum;
        if (whole) {
            stage_out<D, Parts>(stage, a.out, w4 * 32, rows, (job.first + tok) * a.out_stride + (uint64_t)head * D);
            if (there && a.lse) a.lse[(uint64_t)(job.first + tok) * a.n_kv * a.group + head] = lse_of(highest, from, total_sum);
        } else {
            __stcg(rec + D * kRowsL + r, from);
            __stcg(rec + (D + 1) * kRowsL + r, total_sum);
            __stcg(rec + (D + 2) * kRowsL + r, highest);
        }
    }
}

template <int D, int Parts>
__global__ void __launch_bounds__(kThreads, 1) paged_tm_kernel(const __grid_constant__ PagedAttnArgs a) {
    using T = Tm<D, Parts>;
    extern __shared__ uint8_t smem_dyn[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    Head &hd = *reinterpret_cast<Head *>(base);
    uint8_t *q_s = base + T::kHead, *ring = q_s + T::kQ;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a.kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a.vmap) : "memory");
        for (uint32_t s = 0; s < T::kSlots; ++s) { mbar_init(&hd.full[s], 1); mbar_init(&hd.empty[s], 1); }
        for (uint32_t s = 0; s < 8; ++s) mbar_init(&hd.v_ready[s], 1);
        for (int l = 0; l < 2; ++l) { mbar_init(&hd.s_full[l], 1); mbar_init(&hd.p_full[l][0], 4); mbar_init(&hd.p_full[l][1], 4); mbar_init(&hd.o_done[l], 1); }
        mbar_init(&hd.q_full, 8);
        mbar_init(&hd.drain, 1);
        hd.abort_flag = 0;
        hd.any_unfinite = 0;
        fence_barrier_init();
    }
    griddep_wait();
    if (tid == 0) {
        a.blocks[blockIdx.x].records = 0;
        records_left(a)[2 * blockIdx.x] = records_left(a)[2 * blockIdx.x + 1] = 0;
    }

    // ---- this CTA's share of the line: every warp by itself for up to 32 sequences ----
    Shares sh;
    Walk walk;
    Piece p;
    bool bad = false;
    if (a.n_seq <= 32) {
        const PagedSeq q = lane < a.n_seq ? paged_seq(a, lane, bad) : PagedSeq{0, 0, 0};
        const uint32_t few = few_limit(a, q);
        const uint64_t mine = head_units(a, few, q, lane) * a.n_kv;
        const bool fits = __reduce_add_sync(0xffffffffu, (uint32_t)min(mine >> 16, (uint64_t)0x10000u) + 1u) <= 0x10000u;   // (then all of them stay below 2^32)
        bad |= !fits;
        const uint32_t u = fits ? (uint32_t)mine : 0u;
        uint32_t x = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        if (bad && blockIdx.x == 0) atomicCAS(a.status, ST_OK, ST_PAGED_ARGS);
        sh = tm_shares(__shfl_sync(0xffffffffu, x, 31), gridDim.x);
        walk = Walk{share_lo(sh, blockIdx.x), share_lo(sh, blockIdx.x + 1), few};
        const uint32_t at = __ballot_sync(0xffffffffu, walk.pos < x);   // sequences that end behind the share's begin
        const int src = at ? __ffs(at) - 1 : 0;
        p.seq = src;
        p.q.first = __shfl_sync(0xffffffffu, q.first, src);
        p.q.n = __shfl_sync(0xffffffffu, q.n, src);
        p.q.past = __shfl_sync(0xffffffffu, q.past, src);
        p.base = __shfl_sync(0xffffffffu, x - u, src);
    } else {
        uint64_t total = 0, mine = 0;
        for (uint32_t s0 = 0; s0 < a.n_seq; s0 += kThreads) {
            bool b = false;
            const PagedSeq q = s0 + tid < a.n_seq ? paged_seq(a, s0 + tid, b) : PagedSeq{0, 0, 0};
            bad |= b;
            mine += head_units(a, kFewRows, q, lane) * a.n_kv;   // (more than 32 sequences: each by its rows)
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0) hd.sum[warp] = mine;
        __syncthreads();
        for (uint32_t w = 0; w < kThreads / 32; ++w) total += hd.sum[w];
        if ((bad || total >> 32) && blockIdx.x == 0) atomicCAS(a.status, ST_OK, ST_PAGED_ARGS);
        sh = tm_shares(total >> 32 ? 0u : (uint32_t)total, gridDim.x);
        walk = Walk{share_lo(sh, blockIdx.x), share_lo(sh, blockIdx.x + 1), kFewRows};
        uint64_t run = 0;
        for (uint32_t s0 = 0; s0 < a.n_seq && blockIdx.x < sh.n && run <= walk.pos; s0 += kThreads) {
            const PagedSeq q = s0 + tid < a.n_seq ? paged_seq(a, s0 + tid, bad) : PagedSeq{0, 0, 0};
            const uint64_t u = head_units(a, kFewRows, q, lane) * a.n_kv;
            uint64_t x = u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= (uint32_t)o) x += y;
            }
            __syncthreads();
            if (lane == 31) hd.sum[warp] = x;
            __syncthreads();
            x += run - u;
            for (uint32_t w = 0; w < kThreads / 32; ++w) {
                if (w < warp) x += hd.sum[w];
                run += hd.sum[w];
            }
            if (walk.pos >= x && walk.pos < x + u) { hd.start_seq = s0 + tid; hd.start_off = (uint32_t)x; }
        }
        __syncthreads();
        if (blockIdx.x < sh.n) {
            p.seq = hd.start_seq;
            p.base = hd.start_off;
            p.q = paged_seq(a, p.seq, bad);
        }
    }
    if (blockIdx.x >= sh.n) return;
    const bool some = first_piece(a, walk, p) || next_piece(a, walk, p);   // (a share may lie within a block's front)
    __syncthreads();
    for (uint32_t i = tid; i < 3 * D; i += kThreads) hd.unfinite[i] = 0x7fffffffu;
    if (warp == kTensorWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hd.tmem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = hd.tmem;
    bool dead = false;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (!dead && !__all_sync(0xffffffffu, try_bar(bar, parity))) dead = !wait_slow(bar, parity, a.status, &hd.abort_flag);
        return !dead;
    };
    uint32_t done = 0;      // copies of the pieces in front
    uint32_t pieces_in = 0; // pieces begun

    if (warp == kCopyWarp) {
        // ---- copies ----
        const uint32_t box = min(1u << a.page_shift, kTile), boxes = kTile / box, bytes = box * D * 2;
        const uint32_t outside = pool_groups(a.n_pages, a.n_kv, a.page_shift);
        uint32_t issued = 0;
        for (bool more = some; more && !dead; more = next_piece(a, walk, p)) {
            const int32_t *row = a.table + (uint64_t)p.seq * a.max_blocks;
            const uint32_t n = p.t1 - p.t0;
            const bool sm = small(p);
            auto tile_at = [&](uint32_t i, bool &v) { return p.t0 + copy_at(sm, i, n, v); };
            auto page_at = [&](uint32_t tile) -> int32_t {
                const uint32_t key = tile * kTile + lane * box;
                return lane < boxes && key < (uint32_t)p.b.keys ? row[key >> a.page_shift] : -1;
            };
            bool v;
            int32_t page = page_at(tile_at(0, v));
            for (uint32_t i = 0; i < 2 * n; ++i) {
                const uint32_t tile = tile_at(i, v), key = tile * kTile + lane * box, slot = (done + i) % T::kSlots, par = ((done + i) / T::kSlots) & 1u;
                uint32_t at = outside;   // copies from there bring zeros
                if (lane < boxes && key < (uint32_t)p.b.keys) {
                    if (page_there(page, a.n_pages)) at = page_group((uint32_t)page, a.n_kv, p.hkv, a.page_shift, key);
                    else atomicCAS(a.status, ST_OK, ST_PAGED_PAGE);
                }
                bool v2;
                if (i + 1 < 2 * n) page = page_at(tile_at(i + 1, v2));
                if (!wait(&hd.empty[slot], par ^ 1u)) break;
                if (lane == 0) mbar_arrive_expect_tx(&hd.full[slot], T::kPart);
                __syncwarp();
                if (lane < boxes) {
                    const CUtensorMap *map = v ? &a.vmap : &a.kmap;
                    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3}], [%4];" ::"r"(
                                     smem_u32(ring) + slot * T::kPart + lane * bytes),
                                 "l"(map), "r"(0u), "r"(at), "r"(smem_u32(&hd.full[slot])) : "memory");
                }
                issued = done + i + 1;
            }
            done += 2 * n;
        }
        if (dead)   // nothing in flight when the shared memory goes back
            for (uint32_t s = 0; s < T::kSlots; ++s)
                if (issued > s) {
                    const uint32_t last = (issued - 1 - s) / T::kSlots;   // the slot's last use
                    const uint64_t t0 = globaltimer_ns();
                    while (!try_bar(&hd.full[s], last & 1u) && globaltimer_ns() - t0 < kDefaultWaitNs) {}
                }
    } else if (warp == kTensorWarp) {
        // ---- tensor cores ----
        constexpr uint32_t kIdS = idesc_of(kTile, false), kIdO = idesc_of(D, true), kGroup = D * 16;
        uint32_t pv[2] = {0, 0};   // PV products of a lane so far
        uint32_t v_done = 0;       // V tiles of the pieces in front
        const uint32_t ring_s = smem_u32(ring);
        const uint64_t q_desc = desc(smem_u32(q_s), 0, 1024), k_desc = desc(ring_s, 0, kGroup), v_desc = desc(ring_s, 1024, kGroup);
        // A copy's slot and the parity of its barrier. (Waits for several barriers ask for all of them before they look at an answer: one
        // round trip to shared memory instead of one each; the tensor cores stand still meanwhile.)
        auto slot_of = [&](uint32_t i) { return (done + i) % T::kSlots; };
        auto parity_of = [&](uint32_t i) { return ((done + i) / T::kSlots) & 1u; };
        auto wait2 = [&](uint64_t *x, uint32_t px, uint64_t *y, uint32_t py) {
            const bool gx = try_bar(x, px), gy = try_bar(y, py);
            return __all_sync(0xffffffffu, gx && gy) || (wait(x, px) && wait(y, py));
        };
        auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
        auto scores = [&](uint32_t l, uint32_t ql, uint32_t slot) {   // of lane l, q of lane ql, K in a slot
            const uint32_t d = tmem + l * kTile;
            const uint64_t qd = q_desc + (ql * Parts * T::kPart >> 4), kd = k_desc + (slot * T::kPart >> 4);
            if (elect_one()) {
#pragma unroll
                for (int part = Parts - 1; part >= 0; --part)
#pragma unroll
                    for (int kb = 0; kb < D / 16; ++kb)
                        mma_ss(d, qd + ((part * T::kPart + (kb >> 2) * (kRowsL * 128) + (kb & 3) * 32) >> 4), kd + (((kb >> 2) * 1024 + (kb & 3) * 32) >> 4), kIdS,
                               part != Parts - 1 || kb != 0);
                commit(&hd.s_full[l]);
            }
            __syncwarp();
        };
        // O += P V for keys 64 .. 127 (first), then 0 .. 63 of the tile, V in a slot
        auto context = [&](uint32_t l, uint32_t slot, uint32_t half, bool from_zero) {
            const uint32_t d = tmem + kOCol + l * 128, pa = tmem + l * kTile + half * 64;
            const uint64_t vd = v_desc + ((slot * T::kPart + half * 8 * kGroup) >> 4);
            if (elect_one()) {
#pragma unroll
                for (int part = Parts - 1; part >= 0; --part)
#pragma unroll
                    for (int kk = 0; kk < (int)kTile / 32; ++kk)
                        mma_ts(d, pa + (kk >> 1) * 32 + part * 16 + (kk & 1) * 8, vd + ((kk * 2 * kGroup) >> 4), kIdO, !from_zero || part != Parts - 1 || kk != 0);
                if (!half) commit(&hd.o_done[l]);
            }
            __syncwarp();
        };
        auto release = [&](uint32_t slot) {
            if (elect_one()) commit(&hd.empty[slot]);
            __syncwarp();
        };
        for (bool more = some; more && !dead; more = next_piece(a, walk, p)) {
            const uint32_t n = p.t1 - p.t0;
            const bool sm = small(p);
            if (!wait(&hd.q_full, pieces_in & 1u)) break;
            ++pieces_in;
            fence_after();
            // the first scores
            uint32_t slot = uniform(slot_of(0));
            if (!wait(&hd.full[slot], parity_of(0))) break;
            scores(0, 0, slot);
            if (sm) release(slot);
            if (!sm || n > 1) {
                if (sm) {
                    slot = uniform(slot_of(1));
                    if (!wait(&hd.full[slot], parity_of(1))) break;
                }
                scores(1, sm ? 0 : 1, slot);
                release(slot);
            }
            const uint32_t steps = sm ? (n + 1) / 2 : n;
            for (uint32_t step = 0; step < steps && !dead; ++step)
                for (uint32_t l = 0; l < 2 && !dead; ++l) {
                    const uint32_t t = sm ? 2 * step + l : step, next = sm ? t + 2 : t + 1;
                    if (t >= n) break;
                    // (what the value warp has seen has landed)
                    const uint32_t vs = uniform(slot_of(v_index(sm, t, n))), ki = k_index(sm, next), ks = uniform(slot_of(ki)), v_count = v_done + t;
                    if (!wait2(&hd.p_full[l][1], pv[l] & 1u, &hd.v_ready[v_count & 7u], v_count >> 3 & 1u)) break;
                    fence_after();
                    context(l, vs, 1, step == 0);
                    if (!wait(&hd.p_full[l][0], pv[l] & 1u)) break;
                    fence_after();
                    context(l, vs, 0, false);
                    ++pv[l];
                    if (sm || l == 1) release(vs);
                    if (next < n) {
                        // (the next scores overwrite the probabilities)
                        if (!wait2(&hd.full[ks], parity_of(ki), &hd.o_done[l], (pv[l] - 1) & 1u)) break;
                        fence_after();
                        scores(l, sm ? 0 : l, ks);
                        if (sm || l == 1) release(ks);
                    }
                }
            v_done += n;
            done += 2 * n;
        }
        if (dead) {
            if (elect_one()) commit(&hd.drain);
            __syncwarp();
            const uint64_t t0 = globaltimer_ns();
            while (!try_bar(&hd.drain, 0) && globaltimer_ns() - t0 < kDefaultWaitNs) {}
        }
    } else if (warp == kValueWarp) {
        // ---- values that must not meet the tensor cores ----
        uint32_t v_seen = 0;
        if (some) prefetch_q<D, Parts>(a, p);
        for (bool more = some; more && !dead; more = next_piece(a, walk, p)) {
            const uint32_t n = p.t1 - p.t0;
            const bool sm = small(p);
            if (!wait(&hd.q_full, pieces_in & 1u)) break;   // (the notes of the piece before have been read)
            ++pieces_in;
            {   // the next piece's rows of q to L2
                Walk w2 = walk;
                Piece p2 = p;
                if (next_piece(a, w2, p2)) prefetch_q<D, Parts>(a, p2);
            }
            const int32_t lim_first = p.q.past + (int32_t)(p.blk * 2 * kRowsL / a.group);
            for (uint32_t t = 0; t < n; ++t, ++v_seen) {
                const uint32_t i = done + v_index(sm, t, n), slot = i % T::kSlots;
                // (a slot is not filled again before its V tile has been reported; at most five reports are ahead of the tensor warp, the V
                // tiles of a full ring; first that the slot was free: a copy before it that has not landed yet would leave the barrier one
                // phase behind, where this phase's parity reads as complete)
                if (!wait(&hd.empty[slot], ((i / T::kSlots) & 1u) ^ 1u) || !wait(&hd.full[slot], (i / T::kSlots) & 1u)) break;
                if (!partly(a, p, p.t0 + t)) {
                    if (lane == 0) arrive(&hd.v_ready[v_seen & 7u]);
                    continue;
                }
                uint8_t *vt = ring + slot * T::kPart;
                const int32_t k0 = (int32_t)((p.t0 + t) * kTile);
                const uint32_t r0 = (uint32_t)max(0, lim_first + 1 - k0);   // the first key that not all rows attend
                // 16-byte piece j: of key j / (D / 8)
                auto piece = [&](uint32_t j) {
                    const uint32_t r = j / (D / 8), c = j % (D / 8);
                    return reinterpret_cast<uint4 *>(vt + (r >> 3) * (D * 16) + (c >> 3) * 1024 + (r & 7u) * 128 + (((c ^ r) & 7u) << 4));
                };
                auto ones = [](const uint4 &w) {   // bits 15, 31: an exponent of all ones in a half
                    return ((w.x & 0x7C007C00u) + 0x04000400u) | ((w.y & 0x7C007C00u) + 0x04000400u) | ((w.z & 0x7C007C00u) + 0x04000400u) | ((w.w & 0x7C007C00u) + 0x04000400u);
                };
                const uint32_t end = (uint32_t)min((int32_t)kTile, p.b.keys - k0) * (D / 8);
                for (uint32_t j = end + lane; j < kTile * (D / 8); j += 32) *piece(j) = make_uint4(0, 0, 0, 0);
                uint32_t any = 0, j0 = r0 * (D / 8) + lane;
                for (; j0 + 7 * 32 < end; j0 += 8 * 32) {   // (eight loads in flight; the tensor cores may be waiting)
                    uint4 w[8];
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) w[j] = *piece(j0 + 32 * j);
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) any |= ones(w[j]);
                }
                for (; j0 < end; j0 += 32) any |= ones(*piece(j0));
                if (__any_sync(0xffffffffu, any & 0x80008000u)) {
                    hd.any_unfinite = 1u;
                    for (uint32_t j = r0 * (D / 8) + lane; j < end; j += 32) {
                        uint4 *at = piece(j);
                        const uint32_t r = j / (D / 8), c = j % (D / 8);
                        const int32_t key = k0 + (int32_t)r;
                        if (ones(*at) & 0x80008000u) {
                            __half *h = reinterpret_cast<__half *>(at);
                            for (uint32_t e = 0; e < 8; ++e) {
                                const uint16_t b = __half_as_ushort(h[e]);
                                if ((b & 0x7C00u) == 0x7C00u) {
                                    atomicMin(&hd.unfinite[((b & 0x3FFu) ? 2 : b >> 15) * D + c * 8 + e], (uint32_t)key);
                                    h[e] = __ushort_as_half(0);
                                }
                            }
                        }
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) arrive(&hd.v_ready[v_seen & 7u]);
            }
            done += 2 * n;
        }
    } else {
        // ---- softmax: lane l, thread = row ----
        const uint32_t l = warp >> 2, w4 = warp & 3u, r = tid & 127u;
        const uint32_t ts = tmem + (w4 * 32u << 16) + l * kTile, to = tmem + (w4 * 32u << 16) + kOCol + l * 128;
        float4 *acc_mem = reinterpret_cast<float4 *>(a.part_tm + ((uint64_t)gridDim.x * 4 + blockIdx.x * 2 + l) * T::kRecord) + r;   // this row's sums
        uint32_t s_seen = 0;
        if (warp == 0 && lane == 0) { hd.walk = walk; hd.piece = p; hd.job.slot = some ? 2 : 3; }   // (2: none yet)
        __syncwarp();
        for (;;) {
            if (warp == 0) {
                Walk w = hd.walk;
                Piece x = hd.piece;
                const bool valid = hd.job.slot == 2 || (some && next_piece(a, w, x));
                __syncwarp();
                if (lane == 0) {
                    hd.walk = w;
                    hd.piece = x;
                    Job &j = hd.job;
                    j.valid = valid;
                    if (valid) {
                        const uint32_t c0 = owner_of_tile(sh, x, 0), c1 = owner_of_tile(sh, x, x.b.tiles - 1);
                        j.sm = small(x); j.n = x.t1 - x.t0; j.t0 = x.t0;
                        j.first = x.q.first; j.row0 = x.blk * 2 * kRowsL; j.rows = x.b.rows; j.hkv = x.hkv; j.past = x.q.past;
                        j.whole = c0 == c1;
                        j.slot = j.slot == 2 ? 0 : 1;
                        if (!j.whole && c0 == blockIdx.x) a.blocks[c0] = PagedTmBlock{c1 - c0 + 1, j.slot, j.first, j.row0, j.rows, j.hkv, j.past};
                    }
                }
            }
            bar_both();
            const Job &job = hd.job;
            if (!job.valid) break;
            const bool sm = job.sm;
            const uint32_t t0 = job.t0, row0 = job.row0 + (sm ? 0 : l * kRowsL), rows = min(kRowsL, sm ? job.rows : job.rows - min(job.rows, l * kRowsL));
            const uint32_t steps = sm ? (job.n + 1 - l) / 2 : job.n;
            const uint32_t tok = (row0 + r) / a.group, head = job.hkv * a.group + (row0 + r) - tok * a.group;
            const bool there = r < rows, active = w4 * 32 < rows;
            const int32_t lim = there ? job.past + (int32_t)tok : 0x7fffffff;   // (what a row that is not there comes to stays in it)
            float f = 0.f;
            if (!sm) {
                if (!dead && active) f = load_q<D, Parts>(a, q_s + l * Parts * T::kPart, (job.first + tok) * a.q_stride + (uint64_t)head * D, w4 * 32, rows, false);
            } else {
                // one q for both lanes: 16 rows a warp; the factors by way of memory
                const uint32_t at = job.row0 + warp * 16 + (lane & 15u), t = at / a.group, h = job.hkv * a.group + at - t * a.group;
                float *f_mem = a.part_tm + ((uint64_t)gridDim.x * 4 + blockIdx.x * 2) * T::kRecord + D * kRowsL;
                if (!dead && warp * 16 < rows) {
                    const float mine = load_q<D, Parts>(a, q_s, (job.first + t) * a.q_stride + (uint64_t)h * D, warp * 16, rows, true);
                    if (lane < 16) __stcg(f_mem + warp * 16 + lane, mine);
                }
                bar_both();
                if (active) f = __ldcg(f_mem + r);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) arrive(&hd.q_full);

            float ref = -INFINITY, sum = 0.f, highest = -INFINITY;
            float acc_ref = -INFINITY;                                         // reference of the sums in memory
            uint32_t out_of = 0;                                               // bit c: columns 32 c .. have a sum in memory
            for (uint32_t step = 0; step < steps; ++step) {
                const int32_t k0 = (int32_t)((t0 + (sm ? 2 * step + l : step)) * kTile);
                if (Parts == 2 && active && step >= 2) {
                    // half of O to its sum in memory, while the tensor cores form the scores
                    if (!wait(&hd.o_done[l], (s_seen - 1) & 1u)) break;
                    fence_after();
                    if (out_of == 0) acc_ref = ref;
                    if (ref - acc_ref > 40.f) acc_ref = move_sums(acc_mem, out_of, acc_ref, ref);   // (far below what f32 holds: |O| < 2^47)
                    const float by = ref == acc_ref ? 1.f : exp2_fast(ref - acc_ref);
#pragma unroll 1
                    for (uint32_t c4 = (step & 1u) * (D / 64); c4 < ((step & 1u) + 1) * (D / 64); ++c4) {
                        add_out(to, acc_mem, c4, by, out_of >> c4 & 1u);
                        out_of |= 1u << c4;
                    }
                }
                if (!wait(&hd.s_full[l], s_seen & 1u)) break;
                ++s_seen;
                if (!active) {
                    __syncwarp();
                    if (lane == 0) { arrive(&hd.p_full[l][1]); arrive(&hd.p_full[l][0]); }
                    continue;
                }
                fence_after();
                // The scores come once for the maximum; their last 64 columns stay for the exponentials, the others come again.
                const int32_t valid = lim - k0;   // columns 0 .. valid
                const bool cut = __any_sync(0xffffffffu, valid < (int32_t)kTile - 1);
                float top = -INFINITY, sa[32], sb[32];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    load32(ts + 64 * h, sa);
                    load32(ts + 64 * h + 32, sb);
                    wait_ld(sa);
                    wait_ld(sb);
                    if (cut) {
                        cut_at(sa, valid - 64 * h);
                        cut_at(sb, valid - 64 * h - 32);
                    }
                    top = fmaxf(top, fmaxf(max_of(sa), max_of(sb)));
                }
                const float mx = top * f - kShift;   // -inf: no key
                highest = fmaxf(highest, mx);
                float rescale = 1.f;
                if (mx > ref + (step ? kLag : 0.f)) {   // (-inf + 3 = -inf: the first key of a row sets its reference)
                    const float al = ref == -INFINITY ? 1.f : exp2_fast(ref - mx);
                    ref = mx;
                    sum *= al;
                    rescale = al;
                }
                if (step && (__any_sync(0xffffffffu, rescale != 1.f) || (Parts == 1 && half_goes(step)))) change_o<D, Parts>(a, to, rescale, step, ref);
                const float m = ref == -INFINITY ? 0.f : ref;
                const F2 f2 = pair(f, f), m2 = pair(-m, -m);
                F2 part[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                exp_chunk<Parts>(sa, f2, m2, part, ts + 64);
                load32(ts, sa);
                exp_chunk<Parts>(sb, f2, m2, part, ts + 96);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) arrive(&hd.p_full[l][1]);
                wait_ld(sa);
                load32(ts + 32, sb);
                if (cut) cut_at(sa, valid);
                exp_chunk<Parts>(sa, f2, m2, part, ts);
                wait_ld(sb);
                if (cut) cut_at(sb, valid - 32);
                exp_chunk<Parts>(sb, f2, m2, part, ts + 32);
                float p0, p1, p2, p3;
                unpair(part[0], p0, p1);
                unpair(part[1], p2, p3);
                sum += (p0 + p1) + (p2 + p3);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) arrive(&hd.p_full[l][0]);
            }

            // ---- the piece's results: the rows themselves, or a record ----
            if (steps) {
                // (every PV product of a lane follows one of its scores: as many of both)
                wait(&hd.o_done[l], (s_seen - 1) & 1u);
                fence_after();
                if (Parts == 2) __threadfence();   // (the additions to the sums in memory come before the loads below)
            }
            if (Parts == 1 && active && steps > kOutHalf && !dead) halves_back<D>(a, to, steps, ref);
            finish<D, Parts>(a, hd, q_s, Sums{ref, sum, highest, acc_ref, out_of}, steps != 0 && !dead, tmem);
            fence_before();
            // both lanes are done with q, O and the notes (once a wait has run out the value warp may still be at them: the flag is read once)
            const bool notes = bar_both_any(*static_cast<volatile uint32_t *>(&hd.any_unfinite) != 0);
            if (tid == 0 && !job.whole && !given_up(hd)) records_left(a)[2 * blockIdx.x + job.slot] = 1;
            if (notes) {
                for (uint32_t i = tid; i < 3 * D; i += 256) hd.unfinite[i] = 0x7fffffffu;
                bar_both();
                if (tid == 0) hd.any_unfinite = 0;
            }
        }
    }
    griddep_launch_dependents();
    // every thread comes here, whatever happened; then the tensor memory goes back
    fence_before();
    __syncthreads();
    if (warp == kTensorWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// The rows of the blocks that several CTAs shared: block x is the one that begins in CTA x's share, y 16 of its rows. The records are added in
// order of their CTAs. A launch of its own, so that all SMs read them (one CTA alone: 38 records of 32 rows 97 us).
constexpr uint32_t kCombineRows = 16, kCombineThreads = 128;
template <int D, int Parts>
__global__ void __launch_bounds__(kCombineThreads) paged_tm_combine_kernel(const __grid_constant__ PagedAttnArgs a) {
    __shared__ __align__(16) float4 rows_s[kCombineRows][D / 4 + 1];
    griddep_launch_dependents();
    griddep_wait();
    const PagedTmBlock b = a.blocks[blockIdx.x];
    const uint32_t row0 = blockIdx.y * kCombineRows;
    if (b.records == 0 || row0 >= b.rows) return;
    constexpr uint32_t kRecord = Tm<D, Parts>::kRecord, kChunks = D / 4, kPer = kCombineRows * kChunks / kCombineThreads, kStep = kCombineThreads / kCombineRows;
    const uint32_t rw = threadIdx.x % kCombineRows, c = threadIdx.x / kCombineRows, lane_of = row0 / kRowsL, r = row0 % kRowsL + rw;
    const uint32_t at = b.row0 + row0 + rw, tok = at / a.group, head = b.hkv * a.group + at - tok * a.group;
    const bool there = row0 + rw < b.rows;
    auto record = [&](uint32_t i) { return a.part_tm + (uint64_t)(record_index(blockIdx.x, i, b.slot) * 2 + lane_of) * kRecord; };
    float from = -INFINITY, high = -INFINITY, sum = 0.f;
    uint32_t all = 1;   // (a CTA whose wait ran out left no record: nobody writes)
#pragma unroll 4
    for (uint32_t i = 0; i < b.records; ++i) {
        all &= __ldcg(records_left(a) + record_index(blockIdx.x, i, b.slot));
        from = fmaxf(from, __ldcg(record(i) + D * kRowsL + r));
        high = fmaxf(high, __ldcg(record(i) + (D + 2) * kRowsL + r));
    }
    float4 v[kPer];
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (uint32_t i = 0; i < b.records; ++i) {
        const float *rec = record(i);
        const float m = __ldcg(rec + D * kRowsL + r), x = __ldcg(rec + (D + 1) * kRowsL + r), w = m == -INFINITY ? 0.f : exp2_fast(m - from);
        sum = fmaf(x, w, sum);
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) {
            const float4 u = __ldcg(reinterpret_cast<const float4 *>(rec) + (c + j * kStep) * kRowsL + r);
            v[j].x = fmaf(u.x, w, v[j].x); v[j].y = fmaf(u.y, w, v[j].y); v[j].z = fmaf(u.z, w, v[j].z); v[j].w = fmaf(u.w, w, v[j].w);
        }
    }
    const float inv = b.past + (int32_t)tok < 0 ? 0.f : 1.f / sum;
#pragma unroll
    for (uint32_t j = 0; j < kPer; ++j) rows_s[rw][c + j * kStep] = make_float4(v[j].x * inv, v[j].y * inv, v[j].z * inv, v[j].w * inv);
    if (c == 0 && there && all && a.lse) a.lse[(uint64_t)(b.first + tok) * a.n_kv * a.group + head] = lse_of(high, from, sum);
    __syncthreads();
    if (!all) return;
    for (uint32_t i = threadIdx.x; i < kCombineRows * kChunks; i += kCombineThreads) {
        const uint32_t ro = i / kChunks, ch = i % kChunks;
        if (row0 + ro >= b.rows) break;
        const uint32_t x = b.row0 + row0 + ro, t = x / a.group, h = b.hkv * a.group + x - t * a.group;
        const uint64_t dst = (b.first + t) * a.out_stride + (uint64_t)h * D + ch * 4;
        const float4 y = rows_s[ro][ch];
        if (Parts == 1) *reinterpret_cast<uint2 *>((__half *)a.out + dst) = make_uint2(half2_bits(y.x, y.y), half2_bits(y.z, y.w));
        else *reinterpret_cast<float4 *>((float *)a.out + dst) = y;
    }
}

template <int D, int Parts> constexpr size_t tm_smem() { return Tm<D, Parts>::kBytes + 1024; }
static_assert(tm_smem<128, 2>() <= 227 * 1024 && tm_smem<128, 1>() <= 227 * 1024 && tm_smem<64, 2>() <= 227 * 1024, "shared memory");

const struct { void (*k)(const PagedAttnArgs); size_t smem; void (*combine)(const PagedAttnArgs); } kKernels[2][2] = {
    {{paged_tm_kernel<64, 2>, tm_smem<64, 2>(), paged_tm_combine_kernel<64, 2>}, {paged_tm_kernel<64, 1>, tm_smem<64, 1>(), paged_tm_combine_kernel<64, 1>}},
    {{paged_tm_kernel<128, 2>, tm_smem<128, 2>(), paged_tm_combine_kernel<128, 2>}, {paged_tm_kernel<128, 1>, tm_smem<128, 1>(), paged_tm_combine_kernel<128, 1>}}};

} // namespace

cudaError_t paged_tm_init(void) {
    for (const auto &row : kKernels)
        for (const auto &k : row)
            if (const cudaError_t e = cudaFuncSetAttribute(k.k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem)) return e;
    return cudaSuccess;
}

size_t paged_tm_part_bytes(int sms) { return (size_t)6 * sms * Tm<128, 2>::kRecord * sizeof(float) + (size_t)sms * (sizeof(PagedTmBlock) + 2 * sizeof(uint32_t)); }

cudaError_t launch_paged_tm(PagedAttnArgs a, const void *k, const void *v, uint32_t head_dim, int sms, cudaStream_t stream) {
    const uint64_t rows = (uint64_t)a.n_pages * a.n_kv << a.page_shift;
    const uint32_t box = std::min(1u << a.page_shift, kTile);
    a.blocks = reinterpret_cast<PagedTmBlock *>(a.part_tm + (size_t)6 * sms * Tm<128, 2>::kRecord);
    if (const cudaError_t e = tensor_map_groups_swz(&a.kmap, k, rows, head_dim, box)) return e;
    if (const cudaError_t e = tensor_map_groups_swz(&a.vmap, v, rows, head_dim, box)) return e;
    const auto &kernel = kKernels[head_dim == 128][a.half];
    if (const cudaError_t e = launch_kernel(kernel.k, dim3((uint32_t)sms), dim3(kThreads), kernel.smem, stream, true, a)) return e;
    return launch_kernel(kernel.combine, dim3((uint32_t)sms, 2 * kRowsL / kCombineRows), dim3(kCombineThreads), 0, stream, true, a);
}

} // namespace flb
