// Attention over a paged cache, many rows per sequence and KV head (prompt chunks, drafts): blocks of up to 256 rows (token,
// query head of the group) against tiles of 128 keys on tcgen05, scores and contexts in tensor memory.
//
// The mathematics are attn_paged.cu's: an online softmax in f32. f32 activations: q and the probabilities are two f16 parts each, so
// that a pair of row and key costs 8 D tensor flops instead of 4 D, and nothing else is rounded below 32 bits. f16
// activations (Parts = 1): q as it is, the probabilities as one f16 (half a step of 2^-11, as the result).
//
// Bound by the tensor cores. Roles of a CTA (12 warps, one CTA per SM):
//   softmax (2 x 4 warps): "lane" l = its 128 rows, thread = row: scores out of tensor memory, maximum, exponentials, probabilities
//                          back over the scores' columns; at the end of a piece the contexts out
//   copy    (1 warp)     : K and V tiles into a ring of slots, one TMA box per page (attn_paged.cu)
//   tensor  (1 warp)     : scores S = Q K^T (Q, K in shared memory), context O += P V (P in tensor memory)
//   values  (1 warp)     : V tiles that hold keys which only part of the rows attend: keys behind the last are cleared, values that
//                          are not finite are taken out and noted (0 x NaN; see unfinite_of)
// While one lane's softmax runs the tensor cores work for the other: a block of more than 128 rows gives each lane 128 of them over the same
// tiles; a smaller block gives both lanes its rows, every other tile each, and their results are added as two records.
// Tiles of all blocks lie on one line (sequence, KV head, block, tile); shares, records and tickets as in attn_paged.cu.
//
// The tensor cores truncate their running sum, 1.3e-8 of it per instruction; with f32 activations O is therefore
// brought out and added in f32 every kFlush tiles (128 instructions), into a buffer of the CTA's own that stays in L2.
#include "common.cuh"
#include "paged.h"

#include <algorithm>

namespace flb {

namespace {

constexpr uint32_t kRowsL = 128, kTile = 128, kFlush = 8;
constexpr uint32_t kCopyWarp = 8, kTensorWarp = 9, kValueWarp = 10, kThreads = 12 * 32;   // (the last warp completes a warpgroup)
// Registers: 168 a thread at launch; the softmax warps hold a row of 128 scores. 128 (208 + 208 + 88) = 384 x 168.
constexpr uint32_t kRegsSoftmax = 208, kRegsOther = 88;
constexpr float kShift = 6.f;   // probabilities are 2^(x - ref), ref = maximum - 6 when it is set and kept while they stay below 2^14
constexpr uint32_t kOCol = 256, kTmemCols = 512;

template <int D, int Parts> struct Tm {
    static constexpr uint32_t kPart = kRowsL * D * 2;               // one part of a lane's q; a K or V tile
    static constexpr uint32_t kQ = 2 * Parts * kPart;
    static constexpr uint32_t kSlots = D == 64 ? 8 : Parts == 2 ? 3 : 5;
    static constexpr uint32_t kHead = 2048;                         // barriers and the like, in front
    static constexpr uint32_t kBytes = kHead + kQ + kSlots * kPart;
    static constexpr uint32_t kRecord = kRowsL * (D + 3);           // floats: [D / 4][128 rows][4], then references, sums, maxima
};
struct Head {
    uint64_t full[8], empty[8], ready[8], s_full[2], p_full[2], o_done[2], q_full, drain;
    uint64_t total, start_off, sum[kThreads / 32];
    uint32_t start_seq, tmem, abort_flag, last[2], ticket;
    uint32_t unfinite[3 * 128];
};
static_assert(sizeof(Head) <= 2048, "head");

__device__ __forceinline__ float unfinite_at(const uint32_t *u, uint32_t dims, uint32_t d, int32_t lim) {   // attn_paged.cu's unfinite_of
    const int32_t p = (int32_t)u[d], n = (int32_t)u[dims + d], x = (int32_t)u[2 * dims + d];
    if (x <= lim || (p <= lim && n <= lim)) return __int_as_float(0x7fffffff);
    return p <= lim ? INFINITY : n <= lim ? -INFINITY : 0.f;
}

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

// ---- blocks, shares, pieces --------------------------------------------------------------------------------------------
struct Block { uint32_t rows, tiles; int32_t keys; };
__device__ __forceinline__ Block block_of(const PagedAttnArgs &a, const PagedSeq &q, uint32_t blk) {
    Block b;
    b.rows = min(2 * kRowsL, q.n * a.group - blk * 2 * kRowsL);
    b.keys = max(0, q.past + (int32_t)((blk * 2 * kRowsL + b.rows - 1) / a.group) + 1);
    b.tiles = max(1u, ((uint32_t)b.keys + kTile - 1) / kTile);
    return b;
}
__device__ __forceinline__ uint32_t blocks_of(const PagedAttnArgs &a, const PagedSeq &q) {   // of this kernel: sequences of more than few_rows rows
    const uint32_t rows = q.n * a.group;
    return rows > a.few_rows ? (rows + 2 * kRowsL - 1) / (2 * kRowsL) : 0u;
}
// Tiles of every lane's sequence over one KV head; long ones are summed by the whole warp.
__device__ __forceinline__ uint64_t head_units(const PagedAttnArgs &a, const PagedSeq &q, uint32_t lane) {
    const uint32_t n = blocks_of(a, q);
    uint64_t u = 0;
    if (n <= 4)
        for (uint32_t b = 0; b < n; ++b) u += block_of(a, q, b).tiles;
    for (uint32_t todo = __ballot_sync(0xffffffffu, n > 4); todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        PagedSeq x;
        x.first = 0;
        x.n = __shfl_sync(0xffffffffu, q.n, src);
        x.past = __shfl_sync(0xffffffffu, q.past, src);
        const uint32_t nb = __shfl_sync(0xffffffffu, n, src);
        uint64_t v = 0;
        for (uint32_t b = lane; b < nb; b += 32) v += block_of(a, x, b).tiles;
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == (uint32_t)src) u = v;
    }
    return u;
}

struct Piece {
    PagedSeq q;
    uint32_t seq, hkv, blk, n_blk;
    Block b;
    uint32_t t0, t1;
    uint64_t base;       // unit of its block's tile 0
};
struct Walk {
    uint64_t pos, hi, seq_base;
    uint32_t seq;
    bool fresh;
};
// The next piece of a CTA's share, for a whole warp.
__device__ __forceinline__ bool next_piece(const PagedAttnArgs &a, Walk &w, Piece &p) {
    if (w.pos >= w.hi) return false;
    bool bad;
    if (w.fresh) {
        w.fresh = false;
        p.seq = w.seq;
        p.q = paged_seq(a, p.seq, bad);
        p.n_blk = blocks_of(a, p.q);
        // the KV head, then the block (32 at a time), that hold the share's first unit
        const uint32_t lane = threadIdx.x & 31u;
        uint64_t per_head = 0;
        for (uint32_t b = lane; b < p.n_blk; b += 32) per_head += block_of(a, p.q, b).tiles;
#pragma unroll
        for (int o = 16; o; o >>= 1) per_head += __shfl_xor_sync(0xffffffffu, per_head, o);
        p.hkv = (uint32_t)((w.pos - w.seq_base) / per_head);
        p.base = w.seq_base + p.hkv * per_head;
        for (uint32_t b0 = 0;; b0 += 32) {
            const uint64_t t = b0 + lane < p.n_blk ? block_of(a, p.q, b0 + lane).tiles : 0u;
            uint64_t x = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
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
    } else {
        p.base += p.b.tiles;
        if (++p.blk == p.n_blk) {
            p.blk = 0;
            if (++p.hkv == a.n_kv) {
                p.hkv = 0;
                do { p.q = paged_seq(a, ++p.seq, bad); } while ((p.n_blk = blocks_of(a, p.q)) == 0);
            }
        }
        p.b = block_of(a, p.q, p.blk);
    }
    p.t0 = (uint32_t)(w.pos - p.base);
    p.t1 = (uint32_t)min((uint64_t)p.b.tiles, w.hi - p.base);
    w.pos += p.t1 - p.t0;
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

template <int D, int Parts>
__global__ void __launch_bounds__(kThreads, 1) paged_tm_kernel(const __grid_constant__ PagedAttnArgs a) {
    using T = Tm<D, Parts>;
    extern __shared__ uint8_t smem_dyn[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    Head &hd = *reinterpret_cast<Head *>(base);
    uint8_t *q_s = base + T::kHead, *ring = q_s + T::kQ;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    if (tid == 0) {
        for (uint32_t s = 0; s < T::kSlots; ++s) { mbar_init(&hd.full[s], 1); mbar_init(&hd.empty[s], 1); mbar_init(&hd.ready[s], 1); }
        for (int l = 0; l < 2; ++l) { mbar_init(&hd.s_full[l], 1); mbar_init(&hd.p_full[l], 4); mbar_init(&hd.o_done[l], 1); }
        mbar_init(&hd.q_full, 8);
        mbar_init(&hd.drain, 1);
        hd.abort_flag = 0;
        hd.ticket = 0;
        fence_barrier_init();
    }
    for (uint32_t i = tid; i < 3 * D; i += kThreads) hd.unfinite[i] = 0x7fffffffu;
    griddep_wait();

    // ---- this CTA's share of the line ----
    uint64_t total = 0;
    {
        bool bad = false, any_bad = false;
        uint64_t mine = 0;
        for (uint32_t s0 = 0; s0 < a.n_seq; s0 += kThreads) {
            const PagedSeq q = s0 + tid < a.n_seq ? paged_seq(a, s0 + tid, bad) : PagedSeq{0, 0, 0};
            any_bad |= bad;
            mine += head_units(a, q, lane) * a.n_kv;
        }
        if (any_bad && blockIdx.x == 0) atomicCAS(a.status, ST_OK, ST_PAGED_ARGS);
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0) hd.sum[warp] = mine;
        __syncthreads();
        for (uint32_t w = 0; w < kThreads / 32; ++w) total += hd.sum[w];
    }
    const uint32_t ctas = (uint32_t)min((uint64_t)gridDim.x, total);
    if (blockIdx.x >= ctas) return;
    const uint64_t lo = share_of(total, ctas, blockIdx.x), hi = share_of(total, ctas, blockIdx.x + 1);
    {
        uint64_t run = 0;
        for (uint32_t s0 = 0; s0 < a.n_seq && run <= lo; s0 += kThreads) {
            bool bad;
            const PagedSeq q = s0 + tid < a.n_seq ? paged_seq(a, s0 + tid, bad) : PagedSeq{0, 0, 0};
            const uint64_t u = head_units(a, q, lane) * a.n_kv;
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
            if (lo >= x && lo < x + u) { hd.start_seq = s0 + tid; hd.start_off = x; }
        }
    }
    if (warp == kTensorWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hd.tmem)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = hd.tmem;
    Walk walk{lo, hi, hd.start_off, hd.start_seq, true};
    Piece p;
    bool dead = false;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (!dead && !__all_sync(0xffffffffu, try_bar(bar, parity))) dead = !wait_slow(bar, parity, a.status, &hd.abort_flag);
        return !dead;
    };
    uint32_t done = 0;      // copies of the pieces in front
    uint32_t pieces_in = 0; // pieces begun

    if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    if (warp == kCopyWarp) {
        // ---- copies ----
        const uint32_t box = min(1u << a.page_shift, kTile), boxes = kTile / box, bytes = box * D * 2;
        const uint32_t page_groups = (1u << a.page_shift) >> 3, outside = a.n_pages * a.n_kv * page_groups;
        uint32_t issued = 0;
        while (!dead && next_piece(a, walk, p)) {
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
                    if ((uint32_t)page < a.n_pages) at = ((uint32_t)page * a.n_kv + p.hkv) * page_groups + ((key & ((1u << a.page_shift) - 1u)) >> 3);
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
        auto ring_wait = [&](uint32_t i) { return wait(&hd.full[(done + i) % T::kSlots], ((done + i) / T::kSlots) & 1u); };
        auto scores = [&](uint32_t l, uint32_t ql, uint32_t i) {   // of lane l, q of lane ql, K in copy i
            const uint32_t d = tmem + l * kTile, qa = smem_u32(q_s) + ql * Parts * T::kPart, ka = smem_u32(ring) + ((done + i) % T::kSlots) * T::kPart;
            if (elect_one()) {
#pragma unroll
                for (int part = Parts - 1; part >= 0; --part)
#pragma unroll
                    for (int kb = 0; kb < D / 16; ++kb)
                        mma_ss(d, desc(qa + part * T::kPart + (kb >> 2) * (kRowsL * 128) + (kb & 3) * 32, 0, 1024), desc(ka + (kb >> 2) * 1024 + (kb & 3) * 32, 0, kGroup), kIdS,
                               part != Parts - 1 || kb != 0);
                commit(&hd.s_full[l]);
            }
            __syncwarp();
        };
        auto context = [&](uint32_t l, uint32_t i, bool from_zero) {   // O += P V, V in copy i
            const uint32_t d = tmem + kOCol + l * 128, pa = tmem + l * kTile, va = smem_u32(ring) + ((done + i) % T::kSlots) * T::kPart;
            if (elect_one()) {
#pragma unroll
                for (int part = Parts - 1; part >= 0; --part)
#pragma unroll
                    for (int kk = 0; kk < (int)kTile / 16; ++kk)
                        mma_ts(d, pa + part * 64 + kk * 8, desc(va + kk * 2 * kGroup, 1024, kGroup), kIdO, !from_zero || part != Parts - 1 || kk != 0);
                commit(&hd.o_done[l]);
            }
            __syncwarp();
            ++pv[l];
        };
        auto ready = [&](uint32_t i) { return wait(&hd.ready[(done + i) % T::kSlots], ((done + i) / T::kSlots) & 1u); };
        auto release = [&](uint32_t i) {
            ready(i);   // (a slot is not filled again before the value warp has seen it; it is long past)
            if (elect_one()) commit(&hd.empty[(done + i) % T::kSlots]);
            __syncwarp();
        };
        while (!dead && next_piece(a, walk, p)) {
            const uint32_t n = p.t1 - p.t0;
            const bool sm = small(p);
            if (!wait(&hd.q_full, pieces_in & 1u)) break;
            ++pieces_in;
            fence_after();
            // the first scores
            if (!ring_wait(0)) break;
            scores(0, 0, 0);
            if (sm) release(0);
            if (!sm || n > 1) {
                const uint32_t i = sm ? 1 : 0;
                if (!ring_wait(i)) break;
                scores(1, sm ? 0 : 1, i);
                release(i);
            }
            const uint32_t steps = sm ? (n + 1) / 2 : n;
            for (uint32_t step = 0; step < steps && !dead; ++step)
                for (uint32_t l = 0; l < 2 && !dead; ++l) {
                    const uint32_t t = sm ? 2 * step + l : step, next = sm ? t + 2 : t + 1;
                    if (t >= n) break;
                    const uint32_t vi = v_index(sm, t, n), ki = k_index(sm, next);
                    if (!ring_wait(vi) || !ready(vi)) break;
                    if (!wait(&hd.p_full[l], pv[l] & 1u)) break;
                    fence_after();
                    context(l, vi, step == 0 || (Parts == 2 && step % kFlush == 0));
                    if (sm || l == 1) release(vi);
                    if (next < n) {
                        // (the next scores overwrite the probabilities)
                        if (!ring_wait(ki) || !wait(&hd.o_done[l], (pv[l] - 1) & 1u)) break;
                        fence_after();
                        scores(l, sm ? 0 : l, ki);
                        if (sm || l == 1) release(ki);
                    }
                }
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
        while (!dead && next_piece(a, walk, p)) {
            const uint32_t n = p.t1 - p.t0;
            const bool sm = small(p);
            if (!wait(&hd.q_full, pieces_in & 1u)) break;   // (the notes of the piece before have been read)
            ++pieces_in;
            const int32_t lim_first = p.q.past + (int32_t)(p.blk * 2 * kRowsL / a.group);
            for (uint32_t i = 0; i < 2 * n; ++i) {
                bool v;
                const uint32_t t = copy_at(sm, i, n, v), slot = (done + i) % T::kSlots;
                if (!wait(&hd.full[slot], ((done + i) / T::kSlots) & 1u)) break;
                if (!v || !partly(a, p, p.t0 + t)) {
                    if (lane == 0) arrive(&hd.ready[slot]);
                    continue;
                }
                uint8_t *vt = ring + slot * T::kPart;
                const int32_t k0 = (int32_t)((p.t0 + t) * kTile);
                const uint32_t r0 = (uint32_t)max(0, lim_first + 1 - k0);   // the first key that not all rows attend
                for (uint32_t j = r0 * (D / 8) + lane; j < kTile * (D / 8); j += 32) {
                    const uint32_t r = j / (D / 8), c = j % (D / 8);
                    const int32_t key = k0 + (int32_t)r;
                    uint4 *at = reinterpret_cast<uint4 *>(vt + (r >> 3) * (D * 16) + (c >> 3) * 1024 + (r & 7u) * 128 + (((c ^ r) & 7u) << 4));
                    if (key >= p.b.keys) {
                        *at = make_uint4(0, 0, 0, 0);
                    } else {
                        const uint4 w = *at;
                        const uint32_t z = ((w.x & 0x7C007C00u) + 0x04000400u) | ((w.y & 0x7C007C00u) + 0x04000400u) | ((w.z & 0x7C007C00u) + 0x04000400u) | ((w.w & 0x7C007C00u) + 0x04000400u);
                        if (z & 0x80008000u) {   // an exponent of all ones
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
                if (lane == 0) arrive(&hd.ready[slot]);
            }
            done += 2 * n;
        }
    } else if (warp < 8) {
        // ---- softmax: lane l, thread = row ----
        const uint32_t l = warp >> 2, w4 = warp & 3u, r = tid & 127u;
        const uint32_t ts = tmem + (w4 * 32u << 16) + l * kTile, to = tmem + (w4 * 32u << 16) + kOCol + l * 128;
        auto bar_lane = [&] {
            if (l) asm volatile("bar.sync 3, 128;" ::: "memory");
            else asm volatile("bar.sync 2, 128;" ::: "memory");
        };
        auto bar_both = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        float *acc_mem = a.part_tm + ((uint64_t)gridDim.x * 4 + blockIdx.x * 2 + l) * T::kRecord;   // this lane's sums (see kFlush)
        uint32_t s_seen = 0;
        bool first = true;
        while (next_piece(a, walk, p)) {
            const bool sm = small(p);
            const uint32_t n = p.t1 - p.t0, row0 = p.blk * 2 * kRowsL + (sm ? 0 : l * kRowsL), rows = min(kRowsL, sm ? p.b.rows : p.b.rows - min(p.b.rows, l * kRowsL));
            // q as f16 parts into shared memory, every row times a power of two that brings its largest value to [2^11, 2^12)
            float f = 0.f;
            if (!dead) {
                uint8_t *qd = q_s + (sm ? 0 : l) * Parts * T::kPart;
                constexpr int V = D / 32;   // values of a thread
#pragma unroll 4
                for (uint32_t i = 0; i < 32; ++i) {
                    const uint32_t rr = w4 * 32 + i, at = row0 + rr, tok = at / a.group, head = p.hkv * a.group + at - tok * a.group;
                    float x[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) x[j] = 0.f;
                    if (rr < rows) {
                        const uint64_t src = (p.q.first + tok) * a.q_stride + (uint64_t)head * D + lane * V;
                        if (a.half) {
#pragma unroll
                            for (int j = 0; j < V; j += 2) {
                                const float2 y = __half22float2(*reinterpret_cast<const __half2 *>((const __half *)a.q + src + j));
                                x[j] = y.x; x[j + 1] = y.y;
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < V; j += 2) {
                                const float2 y = *reinterpret_cast<const float2 *>((const float *)a.q + src + j);
                                x[j] = y.x; x[j + 1] = y.y;
                            }
                        }
                    }
                    float top = 0.f;
#pragma unroll
                    for (int j = 0; j < V; ++j) top = fmaxf(top, fabsf(x[j]));
                    top = warp_max(top);
                    const int e = min(100, max(-100, 138 - (int)(__float_as_uint(top) >> 23)));
                    const float up = __uint_as_float((uint32_t)(e + 127) << 23);
                    if (lane == i) f = fmaxf(a.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - e) << 23), 1e-37f);
                    if (!sm || l == 0) {
                        const uint32_t d0 = lane * V;
                        uint8_t *dst = qd + (d0 >> 6) * (kRowsL * 128) + (rr >> 3) * 1024 + (rr & 7u) * 128 + (((((d0 & 63u) >> 3) ^ rr) & 7u) << 4) + (d0 & 7u) * 2;
#pragma unroll
                        for (int j = 0; j < V; j += 2) {
                            const float u0 = x[j] * up, u1 = x[j + 1] * up;
                            const __half2 h = __floats2half2_rn(u0, u1);
                            *reinterpret_cast<__half2 *>(dst + 2 * j) = h;
                            if (Parts == 2) {
                                const float2 b = __half22float2(h);
                                *reinterpret_cast<uint32_t *>(dst + T::kPart + 2 * j) = half2_bits(u0 - b.x, u1 - b.y);
                            }
                        }
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) arrive(&hd.q_full);

            const uint32_t tok = (row0 + r) / a.group, head = p.hkv * a.group + (row0 + r) - tok * a.group;
            const bool there = r < rows;
            const int32_t lim = there ? p.q.past + (int32_t)tok : 0x7fffffff;   // (what a row that is not there comes to stays in it)
            const bool active = w4 * 32 < rows;
            const uint32_t steps = sm ? (n + 1 - l) / 2 : n;
            float ref = -INFINITY, sum = 0.f, acc_ref = -INFINITY, highest = -INFINITY;
            for (uint32_t step = 0; step < steps; ++step) {
                const int32_t k0 = (int32_t)((p.t0 + (sm ? 2 * step + l : step)) * kTile);
                if (!wait(&hd.s_full[l], s_seen & 1u)) break;
                ++s_seen;
                if (!active) {
                    if (lane == 0) arrive(&hd.p_full[l]);
                    continue;
                }
                fence_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) load32(ts + 32 * c, s + 32 * c);
                wait_ld(s);
                if (__any_sync(0xffffffffu, k0 + 127 > lim)) {
                    const int32_t valid = lim - k0;
#pragma unroll
                    for (int c = 0; c < 128; ++c) s[c] = c <= valid ? s[c] : -INFINITY;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 128; c += 8)
#pragma unroll
                    for (int j = 0; j < 4; ++j) top[j] = fmaxf(top[j], fmaxf(s[c + j], s[c + 4 + j]));
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * f - kShift;   // -inf: no key
                highest = fmaxf(highest, mx);
                const bool from_zero = step == 0 || (Parts == 2 && step % kFlush == 0);
                if (Parts == 2 && step && from_zero) {
                    // O of the last kFlush tiles to the sums in memory (the product that completed it precedes these scores)
                    const float keep = acc_ref == -INFINITY ? 0.f : exp2_fast(acc_ref - ref);
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        load32(to + c, o);
                        float4 *at = reinterpret_cast<float4 *>(acc_mem) + (c / 4) * kRowsL + r;
                        if (step > kFlush) {
                            float4 old[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) old[j] = at[j * kRowsL];
                            wait_ld(o);
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                at[j * kRowsL] = make_float4(fmaf(old[j].x, keep, o[4 * j]), fmaf(old[j].y, keep, o[4 * j + 1]), fmaf(old[j].z, keep, o[4 * j + 2]), fmaf(old[j].w, keep, o[4 * j + 3]));
                        } else {
                            wait_ld(o);
#pragma unroll
                            for (int j = 0; j < 8; ++j) at[j * kRowsL] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                        }
                    }
                    acc_ref = ref;
                }
                {
                    const float was = ref;
                    if (from_zero ? mx > ref : mx > ref + 8.f) ref = mx;   // (from zero: nothing in O to bring along)
                    const float al = was == -INFINITY || ref == was ? 1.f : exp2_fast(was - ref);
                    sum *= al;
                    if (!from_zero && __any_sync(0xffffffffu, al != 1.f)) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float o[32];
                            load32(to + c, o);
                            wait_ld(o);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                uint32_t w[16];
#pragma unroll
                                for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(o[16 * h + j] * al);
                                store16(to + c + 16 * h, w);
                            }
                        }
                    }
                }
                const float m = ref == -INFINITY ? 0.f : ref;
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t ph[16], pl[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float e0 = exp2_fast(fmaf(s[32 * c + 2 * j], f, -m)), e1 = exp2_fast(fmaf(s[32 * c + 2 * j + 1], f, -m));
                        part[j & 1] += e0;
                        part[2 + (j & 1)] += e1;
                        const __half2 h = __floats2half2_rn(e0, e1);
                        ph[j] = *reinterpret_cast<const uint32_t *>(&h);
                        if (Parts == 2) {
                            const float2 b = __half22float2(h);
                            pl[j] = half2_bits(e0 - b.x, e1 - b.y);
                        }
                    }
                    store16(ts + 16 * c, ph);
                    if (Parts == 2) store16(ts + 64 + 16 * c, pl);
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) arrive(&hd.p_full[l]);
            }

            // ---- the piece's results: the rows themselves, or a record ----
            const uint32_t c0 = owner_of(total, ctas, p.base), c1 = owner_of(total, ctas, p.base + p.b.tiles - 1), records = (c1 - c0 + 1) * (sm ? 2 : 1);
            const bool whole = records == 1;
            float *rec = a.part_tm + (uint64_t)((blockIdx.x * 2 + (first ? 0 : 1)) * 2 + l) * T::kRecord;
            first = false;
            if (steps && !dead) {
                // (every PV product of a lane follows one of its scores: as many of both)
                wait(&hd.o_done[l], (s_seen - 1) & 1u);
                fence_after();
            }
            auto put = [&](uint64_t to_out, const float4 &v) {
                if (a.half) *reinterpret_cast<uint2 *>((__half *)a.out + to_out) = make_uint2(half2_bits(v.x, v.y), half2_bits(v.z, v.w));
                else *reinterpret_cast<float4 *>((float *)a.out + to_out) = v;
            };
            const uint64_t dst = (p.q.first + tok) * a.out_stride + (uint64_t)head * D;
            auto put_lse = [&](float mx, float from, float to_sum) {
                a.lse[(uint64_t)(p.q.first + tok) * a.n_kv * a.group + head] =
                    mx == -INFINITY ? make_float2(mx, to_sum) : make_float2((mx + kShift) * 0.693147180559945309f, to_sum * exp2_fast(from - mx - kShift));
            };
            if (steps && !dead && active) {
                const float keep = acc_ref == -INFINITY ? 0.f : exp2_fast(acc_ref - ref), inv = lim < 0 ? 0.f : 1.f / sum;
                const bool acc = Parts == 2 && steps > kFlush;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    load32(to + c, o);
                    wait_ld(o);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float4 v = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                        if (acc) {
                            const float4 old = reinterpret_cast<const float4 *>(acc_mem)[(c / 4 + j) * kRowsL + r];
                            v.x = fmaf(old.x, keep, v.x); v.y = fmaf(old.y, keep, v.y); v.z = fmaf(old.z, keep, v.z); v.w = fmaf(old.w, keep, v.w);
                        }
                        const uint32_t d = c + 4 * j;
                        v.x += unfinite_at(hd.unfinite, D, d, lim); v.y += unfinite_at(hd.unfinite, D, d + 1, lim);
                        v.z += unfinite_at(hd.unfinite, D, d + 2, lim); v.w += unfinite_at(hd.unfinite, D, d + 3, lim);
                        if (!whole) __stcg(reinterpret_cast<float4 *>(rec) + (c / 4 + j) * kRowsL + r, v);
                        else if (there) put(dst + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                    }
                }
                if (whole && there && a.lse) put_lse(highest, ref, sum);
            }
            if (!whole) {
                __stcg(rec + D * kRowsL + r, steps ? ref : -INFINITY);
                __stcg(rec + (D + 1) * kRowsL + r, steps ? sum : 0.f);
                __stcg(rec + (D + 2) * kRowsL + r, steps ? highest : -INFINITY);
                __threadfence();
                bar_lane();
                // (a small block that is this CTA's alone has a ticket of its own: the other may already count the CTA's last block)
                uint32_t *ticket = c0 == c1 ? &hd.ticket : &a.tickets[2 * c0 + (sm ? 0 : l)];
                if (r == 0) hd.last[l] = !dead && atomicAdd(ticket, 1u) == records - 1 ? 1u : 0u;
                bar_lane();
                if (hd.last[l] && there) {
                    __threadfence();
                    const bool c0_first = p.base <= share_of(total, ctas, c0);
                    auto record = [&](uint32_t i) -> const float * {   // in order of CTA, then lane
                        const uint32_t ci = sm ? i >> 1 : i, li = sm ? i & 1u : l;
                        return a.part_tm + (uint64_t)(((c0 + ci) * 2 + (ci || c0_first ? 0 : 1)) * 2 + li) * T::kRecord;
                    };
                    float mr = -INFINITY, ms = 0.f, top = -INFINITY;
                    for (uint32_t i = 0; i < records; ++i) mr = fmaxf(mr, __ldcg(record(i) + D * kRowsL + r));
                    for (uint32_t i = 0; i < records; ++i) {
                        const float m = __ldcg(record(i) + D * kRowsL + r);
                        top = fmaxf(top, __ldcg(record(i) + (D + 2) * kRowsL + r));
                        if (m != -INFINITY) ms = fmaf(__ldcg(record(i) + (D + 1) * kRowsL + r), exp2_fast(m - mr), ms);
                    }
                    const float inv = lim < 0 ? 0.f : 1.f / ms;
                    for (int c = 0; c < D / 4; c += 8) {
                        float4 v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (uint32_t i = 0; i < records; ++i) {
                            const float m = __ldcg(record(i) + D * kRowsL + r);
                            if (m == -INFINITY) continue;
                            const float w = exp2_fast(m - mr);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float4 u = __ldcg(reinterpret_cast<const float4 *>(record(i)) + (c + j) * kRowsL + r);
                                v[j].x = fmaf(u.x, w, v[j].x); v[j].y = fmaf(u.y, w, v[j].y); v[j].z = fmaf(u.z, w, v[j].z); v[j].w = fmaf(u.w, w, v[j].w);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) put(dst + 4 * (c + j), make_float4(v[j].x * inv, v[j].y * inv, v[j].z * inv, v[j].w * inv));
                    }
                    if (a.lse) put_lse(top, mr, ms);
                }
                if (r == 0 && hd.last[l]) *ticket = 0;
            }
            fence_before();
            bar_both();   // both lanes are done with q, O and the notes
            for (uint32_t i = tid; i < 3 * D; i += 256) hd.unfinite[i] = 0x7fffffffu;
            bar_both();
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

template <int D, int Parts> constexpr size_t tm_smem() { return Tm<D, Parts>::kBytes + 1024; }
static_assert(tm_smem<128, 2>() <= 227 * 1024 && tm_smem<128, 1>() <= 227 * 1024 && tm_smem<64, 2>() <= 227 * 1024, "shared memory");

const struct { void (*k)(const PagedAttnArgs); size_t smem; } kKernels[2][2] = {
    {{paged_tm_kernel<64, 2>, tm_smem<64, 2>()}, {paged_tm_kernel<64, 1>, tm_smem<64, 1>()}},
    {{paged_tm_kernel<128, 2>, tm_smem<128, 2>()}, {paged_tm_kernel<128, 1>, tm_smem<128, 1>()}}};

} // namespace

cudaError_t paged_tm_init(void) {
    for (const auto &row : kKernels)
        for (const auto &k : row)
            if (const cudaError_t e = cudaFuncSetAttribute(k.k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem)) return e;
    return cudaSuccess;
}

size_t paged_tm_part_bytes(int sms) { return (size_t)6 * sms * Tm<128, 2>::kRecord * sizeof(float); }

cudaError_t launch_paged_tm(PagedAttnArgs a, const void *k, const void *v, uint32_t head_dim, int sms, cudaStream_t stream) {
    const uint64_t rows = (uint64_t)a.n_pages * a.n_kv << a.page_shift;
    const uint32_t box = std::min(1u << a.page_shift, kTile);
    if (2 * (uint32_t)sms > kPagedTickets) return cudaErrorInvalidConfiguration;
    if (const cudaError_t e = tensor_map_groups_swz(&a.kmap, k, rows, head_dim, box)) return e;
    if (const cudaError_t e = tensor_map_groups_swz(&a.vmap, v, rows, head_dim, box)) return e;
    const auto &kernel = kKernels[head_dim == 128][a.half];
    return launch_kernel(kernel.k, dim3((uint32_t)sms), dim3(kThreads), kernel.smem, stream, true, a);
}

} // namespace flb
