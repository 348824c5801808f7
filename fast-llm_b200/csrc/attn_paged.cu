// Attention over a paged cache, few rows per sequence and KV head: up to 16 rows (token, query head of the group) against tiles
// of 64 keys on mma.sync.
//
// o_r = sum_j exp(s_rj - m_r) v_j / sum_j exp(s_rj - m_r), s_rj = scale q_r . k_j, with the running maximum and sum of an online
// softmax in f32. Bound by the HBM bytes of the keys and values: every tile is read once.
//
// CTA = 4 warps and a producer, two CTAs per SM. The producer's lanes each copy one page's part of a tile (one TMA box of up to 64 rows) into
// a ring of three stages of 32 KB; warp w takes keys 16 w .. 16 w + 15 of a tile. All tiles lie on one line (sequence, KV head, tile) and every CTA
// takes an equal piece of it.
//   scores : A = 16 keys (ldmatrix), B = 4 rows of q as (hi, lo) f16 parts, scaled by a power of two per row so that both parts stay
//            normal numbers: lane (g, t) has row t and keys g and g + 8
//   softmax: row maxima over the 8 lanes of a row
//   context: A = V^T (ldmatrix.trans), B = the probabilities as (hi, lo) parts. A tile's product starts from zero and is added in f32
//            with rounding, since the tensor cores truncate their running sum (1.3e-8 of it per instruction: 1e-5 after 800 tiles).
// Keys as rows of A cost 16 instructions per 16 keys and 4 rows; the rows as A cost 64 for any number of them, and a tile then took 1.25 us
// of mma.sync.
// Measured (8 KV heads, groups of 4, head_dim 128): 4 x 65000 keys 149 us (6.4 TB/s; rows as A 187), 16 x 5500 to 8192 keys on pages of 16 rows
// 78 us (5.9 TB/s), one sequence over 1024 keys 9.1 us, of which the host's call takes 8.3. Four tokens of 4 heads a sequence, 16 rows (bound by
// mma.sync and the softmax): 4 x 65000 keys 164 us, 1 x 8000 27 us.
// A masked value never meets the tensor core as it is, since 0 x NaN is NaN: rows behind the last key are cleared in shared
// memory, and among the keys of the new tokens, which not all rows attend, values that are not finite are taken out there and
// their effect added to the rows that do attend them (see unfinite_of).
#include "common.cuh"
#include "paged.h"

#include <algorithm>

namespace flb {

namespace {

constexpr uint32_t kRowsB = kFewRows, kTile = 64, kStages = 3, kWarps = 4, kThreads = (kWarps + 1) * 32;
// Probabilities are 2^(x - m + 12): their lo parts stay normal f16 numbers down to 2^-14 of the largest, below it are held to 2^-37 of that
constexpr float kShift = 12.f;

// Rows of a sequence over one KV head, 0 where it is the other kernel's; its tiles: at least one, so that somebody writes its rows.
__device__ __forceinline__ uint32_t rows_of(const PagedAttnArgs &a, uint32_t few, const PagedSeq &q) { return q.n * a.group > few ? 0u : q.n * a.group; }
__device__ __forceinline__ uint32_t tiles_of(const PagedSeq &q) { return max(1u, ((uint32_t)max(0, q.past + (int32_t)q.n) + kTile - 1) / kTile); }
__device__ __forceinline__ uint64_t units_of(const PagedAttnArgs &a, uint32_t few, const PagedSeq &q) { return rows_of(a, few, q) ? (uint64_t)tiles_of(q) * a.n_kv : 0u; }

// The pieces of a CTA's share: consecutive tiles of one sequence over one KV head.
struct Piece {
    PagedSeq q;
    uint32_t seq, hkv, rows, tiles, t0, t1;        // tiles t0 .. t1 - 1 of `tiles`
    int32_t keys;
    uint32_t base;                                 // unit of its tile 0
};
struct Walk { uint32_t pos, hi, few; };            // the share's units behind the piece; see few_limit
// Tiles of the piece that begins at w.pos, over KV head p.hkv of the sequence in p.
__device__ __forceinline__ void cut_piece(Walk &w, Piece &p) {
    p.t0 = w.pos - p.base;
    p.t1 = min(p.tiles, w.hi - p.base);
    w.pos += p.t1 - p.t0;
}
// The piece behind p.
__device__ __forceinline__ bool next_piece(const PagedAttnArgs &a, Walk &w, Piece &p) {
    if (w.pos >= w.hi) return false;
    p.base += p.tiles;
    if (++p.hkv == a.n_kv) {
        bool bad;
        p.hkv = 0;
        do { p.q = paged_seq(a, ++p.seq, bad); } while ((p.rows = rows_of(a, w.few, p.q)) == 0);
        p.tiles = tiles_of(p.q);
        p.keys = max(0, p.q.past + (int32_t)p.q.n);
    }
    cut_piece(w, p);
    return true;
}

// A sequence over one KV head whose last record was this CTA's.
struct Late {
    PagedSeq q;
    uint32_t hkv, rows, c0, pieces;
};

template <int D> struct FewSmem {
    static constexpr uint32_t kHalfStage = kTile * D * 2;                 // K or V of a tile
    uint8_t ring[kStages][2 * kHalfStage];                                // 1024-byte aligned
    float o[kWarps * kRowsB * 36];                                        // q as operands; the warps' contexts, a part at a time
    float f[kRowsB];                                                      // score -> exponent of 2
    float m[kWarps][kRowsB], l[kWarps][kRowsB];
    uint32_t unfinite[3][D];                                              // see unfinite_of
    uint64_t full[kStages], empty[kStages];
    uint64_t sum[kThreads / 32];
    uint32_t start_seq, start_off, any_unfinite, abort_flag, n_late, c0, pieces;                // c0, pieces: the CTAs of the piece's tiles
    Late late[2];                                                         // (a CTA shares two at most: its first and its last)
};

__device__ __forceinline__ void bar_consumers() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap *m) { asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// D(16 x 8, f32) += A(16 x 16) B(16 x 8)
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// D = A B
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// Part 0 or 1 of (a, b) as two f16 pairs hi + lo
__device__ __forceinline__ uint32_t part2(float a, float b, uint32_t part) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    return part ? half2_bits(a - f.x, b - f.y) : *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void put(const PagedAttnArgs &a, uint64_t to, const float4 &v) {
    if (a.half) *reinterpret_cast<uint2 *>((__half *)a.out + to) = make_uint2(half2_bits(v.x, v.y), half2_bits(v.z, v.w));
    else *reinterpret_cast<float4 *>((float *)a.out + to) = v;
}
__device__ __forceinline__ void put_lse(const PagedAttnArgs &a, uint64_t tok, uint32_t head, float mx, float s) {
    a.lse[tok * a.n_kv * a.group + head] = make_float2(mx * 0.693147180559945309f, s * 0.000244140625f);   // 2^-kShift
}
// 2^(m - top); 0 for a maximum of nothing beside one of something
__device__ __forceinline__ float weight(float m, float top) { return m == -INFINITY && top != -INFINITY ? 0.f : exp2_fast(top == -INFINITY ? 0.f : m - top); }

// The page that a lane's part of a tile lies on; -1: behind the last key.
__device__ __forceinline__ int32_t page_at(const PagedAttnArgs &a, const Piece &p, uint32_t tile) {
    const uint32_t lane = threadIdx.x & 31u, shift = min(a.page_shift, 6u), key = tile * kTile + (lane << shift);
    return lane < kTile >> shift && key < (uint32_t)p.keys ? a.table[(uint64_t)p.seq * a.max_blocks + (key >> a.page_shift)] : -1;
}
// The producer warp: all tiles of the share into the ring, lane i part i of a tile (one page's or less). Pages are looked up a tile ahead.
template <int D>
__device__ __forceinline__ void copy_tiles(const PagedAttnArgs &a, FewSmem<D> &sm, Walk &walk, Piece &p) {
    constexpr uint32_t kKV = FewSmem<D>::kHalfStage;
    const uint32_t lane = threadIdx.x & 31u, shift = min(a.page_shift, 6u), boxes = kTile >> shift;
    const uint32_t behind = pool_groups(a.n_pages, a.n_kv, a.page_shift);
    uint32_t issued = 0, stage = 0, parity = 1;
    bool landed = true;
    do {
        int32_t page = page_at(a, p, p.t0);
#pragma unroll 1
        for (uint32_t tile = p.t0; tile < p.t1; ++tile) {
            const uint32_t key = tile * kTile + (lane << shift);
            uint32_t at = behind;
            if (lane < boxes && key < (uint32_t)p.keys) {
                if (page_there(page, a.n_pages)) at = page_group((uint32_t)page, a.n_kv, p.hkv, a.page_shift, key);
                else atomicCAS(a.status, ST_OK, ST_PAGED_PAGE);
            }
            if (tile + 1 < p.t1) page = page_at(a, p, tile + 1);
            landed = __all_sync(0xffffffffu, mbar_wait_bounded(&sm.empty[stage], parity, a.status));
            if (!landed) break;
            if (lane == 0) mbar_arrive_expect_tx(&sm.full[stage], 2 * kKV);
            __syncwarp();
            if (lane < boxes) {
                const uint32_t dst = smem_u32(sm.ring[stage]) + ((lane * D * 2) << shift), bar = smem_u32(&sm.full[stage]);
                asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3}], [%4];" ::"r"(dst),
                             "l"(&a.kmap), "r"(0u), "r"(at), "r"(bar) : "memory");
                asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3}], [%4];" ::"r"(dst + kKV),
                             "l"(&a.vmap), "r"(0u), "r"(at), "r"(bar) : "memory");
            }
            ++issued;
            if (++stage == kStages) { stage = 0; parity ^= 1u; }
        }
    } while (landed && next_piece(a, walk, p));
    if (!landed)   // nothing in flight when the shared memory goes back
        for (uint32_t i = issued - min(issued, kStages); i < issued; ++i) mbar_wait_bounded(&sm.full[i % kStages], i / kStages & 1u, a.status);
}

// The records of a sequence over one KV head, added in order: of CTA c0 the one of the tiles that begin in its share, of the others the one
// of tiles that began before. This is the launch's tail: its time is round trips to L2, so that as many records as the ring holds, which is
// free by then, are copied into it at once; then their weights, 8 lanes a row, then the contexts. Run once, so out of line. (16 rows, 42
// records: 11 us; loads into registers, 8 at a time, 20.)
template <int D, int B>
__device__ __noinline__ void combine(const PagedAttnArgs &a, FewSmem<D> &sm, const Late late) {
    constexpr uint32_t kRecord = kRowsB * (D + 4), kChunks = D / 4, kThr = kWarps * 32, kItems = 4 * B * kChunks <= kThr ? 1 : 4 * B * kChunks / kThr;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, len = late.rows * (D + 4), wr = tid >> 3;
    const uint32_t at_once = (uint32_t)(sizeof(sm.ring) / sizeof(float)) / len;
    const float *rec = a.part + (uint64_t)late.c0 * 2 * kRecord;   // record i >= 1 at rec + 2 i kRecord
    const float *in = reinterpret_cast<const float *>(sm.ring);
    const uint32_t in_s = smem_u32(sm.ring);
    static_assert(sizeof(sm.ring) / 4 / (D + 4) <= sizeof(sm.o) / 4 && kThr / 8 == kRowsB, "weights");
    float4 v[kItems];
#pragma unroll
    for (uint32_t j = 0; j < kItems; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, sum = 0.f;   // of row wr
    for (uint32_t k0 = 0; k0 < late.pieces; k0 += at_once) {
        const uint32_t n = min(at_once, late.pieces - k0);
        for (uint32_t k = warp; k < n; k += kWarps) {
            const float *from = rec + (k0 + k ? 2 * (k0 + k) * kRecord : kRecord);
            for (uint32_t i = lane * 4; i < len; i += 128)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(in_s + (k * len + i) * 4), "l"(from + i) : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        bar_consumers();
        const float *ml = in + wr * (D + 4) + D;
        float t = top, add = 0.f;
        if (wr < late.rows)
            for (uint32_t k = lane & 7u; k < n; k += 8) t = fmaxf(t, ml[k * len]);
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        const float old = weight(top, t);
        top = t;
        if (wr < late.rows)
            for (uint32_t k = lane & 7u; k < n; k += 8) {
                const float w = weight(ml[k * len], t);
                sm.o[wr * n + k] = w;
                add = fmaf(ml[k * len + 1], w, add);
            }
        add += __shfl_xor_sync(0xffffffffu, add, 1);
        add += __shfl_xor_sync(0xffffffffu, add, 2);
        add += __shfl_xor_sync(0xffffffffu, add, 4);
        sum = fmaf(sum, old, add);
        if (!(lane & 7u)) { sm.f[wr] = old; sm.m[0][wr] = t; sm.l[0][wr] = sum; }
        bar_consumers();
        const float *u[kItems], *w[kItems];
#pragma unroll
        for (uint32_t j = 0; j < kItems; ++j) {
            const uint32_t i = tid + j * kThr, x = min(i / kChunks, late.rows - 1);
            const float by = sm.f[x];
            v[j].x *= by; v[j].y *= by; v[j].z *= by; v[j].w *= by;
            u[j] = in + x * (D + 4) + i % kChunks * 4;
            w[j] = sm.o + x * n;
        }
#pragma unroll 4
        for (uint32_t k = 0; k < n; ++k)
#pragma unroll
            for (uint32_t j = 0; j < kItems; ++j) {
                const float4 y = *reinterpret_cast<const float4 *>(u[j] + k * len);
                const float by = w[j][k];
                v[j].x = fmaf(y.x, by, v[j].x); v[j].y = fmaf(y.y, by, v[j].y); v[j].z = fmaf(y.z, by, v[j].z); v[j].w = fmaf(y.w, by, v[j].w);
            }
        bar_consumers();
    }
#pragma unroll
    for (uint32_t j = 0; j < kItems; ++j) {
        const uint32_t i = tid + j * kThr, rw = i / kChunks, d = i % kChunks * 4;
        if (rw >= late.rows) break;
        const uint32_t tk = rw / a.group, hd = late.hkv * a.group + rw - tk * a.group;
        const float inv = late.q.past + (int32_t)tk < 0 ? 0.f : 1.f / sm.l[0][rw];
        put(a, (late.q.first + tk) * a.out_stride + (uint64_t)hd * D + d, make_float4(v[j].x * inv, v[j].y * inv, v[j].z * inv, v[j].w * inv));
        if (a.lse && d == 0) put_lse(a, late.q.first + tk, hd, sm.m[0][rw], sm.l[0][rw]);
    }
    bar_consumers();   // (another one may follow)
}
// What values that are not finite add to four dimensions of a row
template <int D> __device__ __noinline__ float4 add_unfinite(const uint32_t *u, uint32_t d, int32_t lim, const float4 v) {
    return make_float4(v.x + unfinite_of(u, D, d, lim), v.y + unfinite_of(u, D, d + 1, lim), v.z + unfinite_of(u, D, d + 2, lim), v.w + unfinite_of(u, D, d + 3, lim));
}

// The rows of a piece as the threads hold them: blocks of 4 (at most B), lane (g, t) row t. q as operand: column g = row g / 2, part
// g & 1; dimensions 2t, 2t + 1, 2t + 8, 2t + 9 of every 16; in registers for one block, else it stays in shared memory.
template <int D, int B> struct Rows {
    uint2 q[B == 1 ? D / 16 : 1];
    float o[B][D / 16][2];                 // contexts: dimensions g and g + 8 of every 16
    float f[B], m[B], l[B];                // score -> exponent of 2; maximum, sum
    int32_t lim[B];                        // last key
};

// A warp's 16 keys (from key k0) against N blocks of rows.
template <int D, int B, int N>
__device__ __forceinline__ void tile_step(Rows<D, B> &w, const uint2 *q_s, uint32_t k_s, uint32_t v_s, int32_t k0) {
    constexpr uint32_t kGroupBytes = 8 * D * 2;
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u, mi = lane >> 3, r8 = lane & 7u;
    float sc[N][4];
#pragma unroll
    for (int kb = 0; kb < D / 16; ++kb) {
        uint32_t ka[4];
        ldsm4(k_s + (mi & 1u) * kGroupBytes + (kb >> 2) * 1024 + r8 * 128 + (((2 * (kb & 3) + (mi >> 1)) ^ r8) << 4), ka);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint2 q = B == 1 ? w.q[kb] : q_s[(n * (D / 16) + kb) * 32];
            if (kb == 0) mma_first(sc[n], ka, q.x, q.y);
            else mma(sc[n], ka, q.x, q.y);
        }
    }
    float al[N];
    uint32_t pb[N][2];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const float s0 = k0 + (int32_t)g <= w.lim[n] ? sc[n][0] + sc[n][1] : -INFINITY, s1 = k0 + 8 + (int32_t)g <= w.lim[n] ? sc[n][2] + sc[n][3] : -INFINITY;
        float top = fmaxf(s0, s1);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float mn = fmaxf(w.m[n], top * w.f[n]), ref = (mn == -INFINITY ? 0.f : mn) - kShift;
        al[n] = exp2_fast(w.m[n] - kShift - ref);
        w.m[n] = mn;
        const float p0 = exp2_fast(fmaf(s0, w.f[n], -ref)), p1 = exp2_fast(fmaf(s1, w.f[n], -ref));
        w.l[n] = fmaf(w.l[n], al[n], p0 + p1);   // (this lane's keys)
        // operand: column g = row g / 2, part g & 1; keys 2t, 2t + 1, 2t + 8, 2t + 9
        const uint32_t src = 8 * t + (g >> 1);
        const float a0 = __shfl_sync(0xffffffffu, p0, src), b0 = __shfl_sync(0xffffffffu, p0, src + 4);
        const float a1 = __shfl_sync(0xffffffffu, p1, src), b1 = __shfl_sync(0xffffffffu, p1, src + 4);
        pb[n][0] = part2(a0, b0, g & 1u);
        pb[n][1] = part2(a1, b1, g & 1u);
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
        uint32_t va[4];
        ldsm4t(v_s + (mi >> 1) * kGroupBytes + (dt >> 2) * 1024 + r8 * 128 + (((2 * (dt & 3) + (mi & 1u)) ^ r8) << 4), va);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float d[4];
            mma_first(d, va, pb[n][0], pb[n][1]);
            w.o[n][dt][0] = fmaf(w.o[n][dt][0], al[n], d[0] + d[1]);
            w.o[n][dt][1] = fmaf(w.o[n][dt][1], al[n], d[2] + d[3]);
        }
    }
}

// Block n of a piece's rows of q as operands into shared memory, with the factors of their scores (a warp).
template <int D>
__device__ __forceinline__ void build_q(const PagedAttnArgs &a, FewSmem<D> &sm, const Piece &p, uint32_t n) {
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t row = n * 4 + (g >> 1), tok = row / a.group, head = p.hkv * a.group + row - tok * a.group;
    const uint64_t src = row < p.rows ? (p.q.first + tok) * a.q_stride + (uint64_t)head * D : 0;
    float2 x[D / 8];
    if (a.half) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) x[j] = __half22float2(*reinterpret_cast<const __half2 *>((const __half *)a.q + src + 8 * j + 2 * t));
    } else {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) x[j] = *reinterpret_cast<const float2 *>((const float *)a.q + src + 8 * j + 2 * t);
    }
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) top = fmaxf(top, fmaxf(fabsf(x[j].x), fabsf(x[j].y)));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // a power of two brings the row's largest value to [2^11, 2^12)
    const int e = min(126, max(-116, 138 - (int)(__float_as_uint(top) >> 23)));   // (-116: the largest f32; 2^-126 is a normal one)
    const float up = __uint_as_float((uint32_t)(e + 127) << 23);
    if (t == 0 && !(g & 1u)) sm.f[row] = fmaxf(a.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - e) << 23), 1e-37f);
    uint2 *to = reinterpret_cast<uint2 *>(sm.o) + n * (D / 16) * 32 + lane;
#pragma unroll
    for (int kb = 0; kb < D / 16; ++kb)
        to[kb * 32] = make_uint2(part2(x[2 * kb].x * up, x[2 * kb].y * up, g & 1u), part2(x[2 * kb + 1].x * up, x[2 * kb + 1].y * up, g & 1u));
}
static_assert(kRowsB / 4 * (128 / 16) * 32 * sizeof(uint2) <= sizeof(FewSmem<128>::o), "q");
template <int D, int B>
__device__ __forceinline__ void begin_rows(const PagedAttnArgs &a, const FewSmem<D> &sm, const Piece &p, Rows<D, B> &w) {
    const uint32_t lane = threadIdx.x & 31u, t = lane & 3u;
    if (B == 1)
#pragma unroll
        for (int kb = 0; kb < D / 16; ++kb) w.q[kb] = reinterpret_cast<const uint2 *>(sm.o)[kb * 32 + lane];
#pragma unroll
    for (uint32_t n = 0; n < B; ++n) {
        const uint32_t mine = n * 4 + t;
        w.f[n] = sm.f[mine];
        w.lim[n] = mine < p.rows ? p.q.past + (int32_t)(mine / a.group) : -1;
        w.m[n] = -INFINITY;
        w.l[n] = 0.f;
#pragma unroll
        for (int kb = 0; kb < D / 16; ++kb) w.o[n][kb][0] = w.o[n][kb][1] = 0.f;
    }
}

// (out of line, and by way of memory: in line 4 x 65000 keys with 16 rows went from 164 to 191 us)
template <int D> __device__ __noinline__ void note_ctas(const PagedAttnArgs &a, FewSmem<D> &sm, const Shares sh, uint32_t b, uint32_t e) {
    const uint32_t snap = a.n_seq <= 32 ? kSnap : 0;
    if (sh.each < 2) {
        sm.c0 = owner_of(sh, b);
        sm.pieces = owner_of(sh, e - 1) - sm.c0 + 1;
        return;
    }
    sm.c0 = first_of(sh, snap, b, e);
    sm.pieces = last_of(sh, snap, b, e) - sm.c0 + 1;
}
template <int D, int B>   // at most 4 B rows
__global__ void __launch_bounds__(kThreads, 2) paged_few_kernel(const __grid_constant__ PagedAttnArgs a) {
    extern __shared__ uint8_t smem_dyn[];
    FewSmem<D> &sm = *reinterpret_cast<FewSmem<D> *>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    constexpr uint32_t kKV = FewSmem<D>::kHalfStage, kGroupBytes = 8 * D * 2;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, t = lane & 3u;
    if (tid == 0) {
        prefetch_map(&a.kmap);
        prefetch_map(&a.vmap);
        for (uint32_t s = 0; s < kStages; ++s) { mbar_init(&sm.full[s], 1); mbar_init(&sm.empty[s], kWarps); }
        sm.abort_flag = 0;
        sm.n_late = 0;
        sm.any_unfinite = 0;
        fence_barrier_init();
    }
    for (uint32_t i = tid; i < 3 * D; i += kThreads) (&sm.unfinite[0][0])[i] = 0x7fffffffu;
    __syncthreads();
    griddep_wait();

    // ---- this CTA's share of the line: every warp by itself for up to 32 sequences ----
    Shares sh;
    Piece p;
    Walk walk;
    if (a.n_seq <= 32) {
        bool bad = false;
        const PagedSeq q = lane < a.n_seq ? paged_seq(a, lane, bad) : PagedSeq{0, 0, 0};
        walk.few = few_limit(a, q);
        const uint64_t mine = units_of(a, walk.few, q);
        bad |= mine >> 26 != 0;   // (32 of them stay below 2^32; 2^26 tiles are 2^32 keys)
        const uint32_t u = mine >> 26 ? 0u : (uint32_t)mine;
        uint32_t x = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        if (bad && blockIdx.x == 0) atomicCAS(a.status, ST_OK, ST_PAGED_ARGS);
        sh = few_shares(__shfl_sync(0xffffffffu, x, 31), gridDim.x);
        if (blockIdx.x >= sh.n) return;
        const uint32_t tiles = max(1u, u / a.n_kv);   // (of the lane's sequence over a KV head)
        auto edge = [&](uint32_t c) {
            const uint32_t at = share_lo(sh, c);
            if (!edge_moves(sh, c)) return at;
            const int src = __ffs(__ballot_sync(0xffffffffu, at < x)) - 1;
            const uint32_t n = __shfl_sync(0xffffffffu, tiles, src), b = at - (at - __shfl_sync(0xffffffffu, x - u, src)) % n;
            return snapped(sh, kSnap, at, b, b + n);
        };
        walk.pos = edge(blockIdx.x);
        walk.hi = edge(blockIdx.x + 1);
        const int src = __ffs(__ballot_sync(0xffffffffu, walk.pos < x)) - 1;   // the first sequence that ends behind the share's begin
        p.seq = src;
        p.q.first = __shfl_sync(0xffffffffu, q.first, src);
        p.q.n = __shfl_sync(0xffffffffu, q.n, src);
        p.q.past = __shfl_sync(0xffffffffu, q.past, src);
        p.base = __shfl_sync(0xffffffffu, x - u, src);
    } else {
        const uint32_t per = (a.n_seq + kThreads - 1) / kThreads, s0 = min(tid * per, a.n_seq), s1 = min(s0 + per, a.n_seq);
        uint64_t mine = 0;
        bool bad = false, any_bad = false;
        for (uint32_t s = s0; s < s1; ++s) {
            mine += units_of(a, kFewRows, paged_seq(a, s, bad));
            any_bad |= bad;
        }
        uint64_t x = mine, total = 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t u = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += u;
        }
        if (lane == 31) sm.sum[warp] = x;
        __syncthreads();
        for (uint32_t w = 0; w < kThreads / 32; ++w) {
            if (w < warp) x += sm.sum[w];
            total += sm.sum[w];
        }
        if ((any_bad || total >> 32) && blockIdx.x == 0) atomicCAS(a.status, ST_OK, ST_PAGED_ARGS);
        x -= mine;
        sh = few_shares(total >> 32 ? 0u : (uint32_t)total, gridDim.x);
        if (blockIdx.x >= sh.n) return;
        walk = Walk{share_lo(sh, blockIdx.x), share_lo(sh, blockIdx.x + 1), kFewRows};
        if (walk.pos >= x && walk.pos < x + mine) {
            uint32_t s = s0;
            for (;; ++s) {
                const uint64_t u = units_of(a, kFewRows, paged_seq(a, s, bad));
                if (walk.pos < x + u) break;
                x += u;
            }
            sm.start_seq = s;
            sm.start_off = (uint32_t)x;
        }
        __syncthreads();
        p.seq = sm.start_seq;
        p.base = sm.start_off;
        p.q = paged_seq(a, p.seq, bad);
    }
    p.rows = rows_of(a, walk.few, p.q);
    p.tiles = tiles_of(p.q);
    p.keys = max(0, p.q.past + (int32_t)p.q.n);
    p.hkv = (walk.pos - p.base) / p.tiles;
    p.base += p.hkv * p.tiles;
    cut_piece(walk, p);
    if (warp == kWarps) {
        copy_tiles<D>(a, sm, walk, p);
        return;
    }

    uint32_t stage = 0, parity = 0;   // of the ring
    bool landed = true;   // no wait of this warp has run out
    do {
        for (uint32_t n = warp; n * 4 < p.rows; n += kWarps) build_q<D>(a, sm, p, n);
        if (tid == 0) note_ctas<D>(a, sm, sh, p.base, p.base + p.tiles);
        bar_consumers();
        Rows<D, B> w;
        begin_rows<D, B>(a, sm, p, w);
        const uint2 *q_s = reinterpret_cast<const uint2 *>(sm.o) + lane;
        const int32_t lim_first = p.q.past;   // last key that all rows attend
#pragma unroll 1
        for (uint32_t tile = p.t0; tile < p.t1; ++tile) {
            landed = landed && __all_sync(0xffffffffu, mbar_wait_bounded(&sm.full[stage], parity, a.status));
            const int32_t k0 = (int32_t)(tile * kTile + warp * 16);
            if (landed && k0 < p.keys) {
                const uint32_t k_s = smem_u32(sm.ring[stage]) + warp * 2 * kGroupBytes, v_s = k_s + kKV;
                if (k0 + 16 > lim_first + 1 || k0 + 16 > p.keys) {
                    uint8_t *vrow = sm.ring[stage] + kKV + warp * 2 * kGroupBytes;
#pragma unroll 1
                    for (uint32_t i = lane; i < 16 * D / 8; i += 32) {
                        const uint32_t r = i / (D / 8), c = i % (D / 8);
                        const int32_t key = k0 + (int32_t)r;
                        uint4 *at = reinterpret_cast<uint4 *>(vrow + (r >> 3) * kGroupBytes + (c >> 3) * 1024 + (r & 7u) * 128 + (((c ^ r) & 7u) << 4));
                        if (key >= p.keys) {
                            *at = make_uint4(0, 0, 0, 0);
                        } else if (key > lim_first) {
                            const uint4 x = *at;
                            const uint32_t z = ((x.x & 0x7C007C00u) + 0x04000400u) | ((x.y & 0x7C007C00u) + 0x04000400u) | ((x.z & 0x7C007C00u) + 0x04000400u) | ((x.w & 0x7C007C00u) + 0x04000400u);
                            if (z & 0x80008000u) {   // an exponent of all ones
                                __half *h = reinterpret_cast<__half *>(at);
                                for (uint32_t j = 0; j < 8; ++j) {
                                    const uint16_t b = __half_as_ushort(h[j]);
                                    if ((b & 0x7C00u) == 0x7C00u) {
                                        sm.any_unfinite = 1u;
                                        atomicMin(&sm.unfinite[(b & 0x3FFu) ? 2 : b >> 15][c * 8 + j], (uint32_t)key);
                                        h[j] = __ushort_as_half(0);
                                    }
                                }
                            }
                        }
                    }
                    fence_proxy_async_smem();   // (the next copy into this stage comes after these writes)
                    __syncwarp();
                }
                if (B == 1 || p.rows <= 4) tile_step<D, B, 1>(w, q_s, k_s, v_s, k0);
                else if (B == 2 || p.rows <= 8) tile_step<D, B, (B < 2 ? 1 : 2)>(w, q_s, k_s, v_s, k0);
                else tile_step<D, B, B>(w, q_s, k_s, v_s, k0);
            }
            __syncwarp();
            if (lane == 0) arrive(&sm.empty[stage]);
            if (++stage == kStages) { stage = 0; parity ^= 1u; }
        }
        if (!landed) sm.abort_flag = 1u;   // (everybody goes on to the barriers, nobody writes)

        // ---- the warps' sums, a part of the dimensions at a time ----
        const uint32_t c0 = sm.c0, pieces = sm.pieces;
        const bool whole = pieces == 1;
        float *rec = a.part + (uint64_t)(blockIdx.x * 2 + (p.t0 == 0 ? 1 : 0)) * kRowsB * (D + 4);   // tiles that begin here, or before
#pragma unroll
        for (uint32_t n = 0; n < B; ++n) {
            if (n * 4 >= p.rows) break;
            w.l[n] += __shfl_xor_sync(0xffffffffu, w.l[n], 4);
            w.l[n] += __shfl_xor_sync(0xffffffffu, w.l[n], 8);
            w.l[n] += __shfl_xor_sync(0xffffffffu, w.l[n], 16);
            if (g == 0) { sm.m[warp][n * 4 + t] = w.m[n]; sm.l[warp][n * 4 + t] = w.l[n]; }
        }
        bar_consumers();
#pragma unroll
        for (uint32_t n = 0; n < B; ++n) {   // contexts relative to the largest maximum
            if (n * 4 >= p.rows) break;
            float top = -INFINITY;
#pragma unroll
            for (uint32_t x = 0; x < kWarps; ++x) top = fmaxf(top, sm.m[x][n * 4 + t]);
            const float by = weight(w.m[n], top);
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) { w.o[n][dt][0] *= by; w.o[n][dt][1] *= by; }
        }
        // parts of `wide` dimensions: few rows, wide parts; the thread's row and 4 dimensions of a part. (All parts in line: as a loop
        // with the registers of a part found at run time 4.2 us for 16 rows, now 2.0.)
        constexpr uint32_t row_bits = B == 4 ? 4 : B == 1 && D == 128 ? 2 : 3, wide = 512u >> row_bits, pitch = wide + 4;
        const uint32_t row = tid >> (7 - row_bits), c4 = (tid & ((wide >> 2) - 1u)) * 4;
        const uint32_t tok = row / a.group, head = p.hkv * a.group + row - tok * a.group;
        const int32_t row_lim = p.q.past + (int32_t)tok;
        const uint64_t dst = (p.q.first + tok) * a.out_stride + (uint64_t)head * D;
        float top = -INFINITY, sum = 0.f;
        const bool writes = row < p.rows && !sm.abort_flag, unfinite = sm.any_unfinite != 0;
        if (row < p.rows) {
#pragma unroll
            for (uint32_t x = 0; x < kWarps; ++x) top = fmaxf(top, sm.m[x][row]);
#pragma unroll
            for (uint32_t x = 0; x < kWarps; ++x) sum = fmaf(sm.l[x][row], weight(sm.m[x][row], top), sum);
        }
        const float inv = row_lim < 0 ? 0.f : 1.f / sum;
#pragma unroll
        for (uint32_t d0 = 0; d0 < D; d0 += wide) {
            if (d0) bar_consumers();
#pragma unroll
            for (uint32_t n = 0; n < B; ++n) {
                float *at = sm.o + ((warp << row_bits) + n * 4 + t) * pitch + g;
#pragma unroll
                for (uint32_t dt = 0; dt < wide / 16; ++dt) { at[dt * 16] = w.o[n][d0 / 16 + dt][0]; at[dt * 16 + 8] = w.o[n][d0 / 16 + dt][1]; }
            }
            bar_consumers();
            if (writes) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (uint32_t x = 0; x < kWarps; ++x) {
                    const float4 u = *reinterpret_cast<const float4 *>(&sm.o[((x << row_bits) + row) * pitch + c4]);
                    v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
                }
                const uint32_t d = d0 + c4;
                if (unfinite) v = add_unfinite<D>(&sm.unfinite[0][0], d, row_lim, v);
                if (whole) put(a, dst + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                else __stcg(reinterpret_cast<float4 *>(rec + row * (D + 4) + d), v);
            }
        }
        if (writes && c4 == 0) {
            if (!whole) __stcg(reinterpret_cast<float4 *>(rec + row * (D + 4) + D), make_float4(top, sum, 0.f, 0.f));
            else if (a.lse) put_lse(a, p.q.first + tok, head, top, sum);
        }
        if (!whole) {
            fence_acq_rel_gpu();
            bar_consumers();
            if (tid == 0) {   // (the ticket is the next launch's again whatever became of this one)
                const bool gave_up = sm.abort_flag != 0;
                const uint32_t before = atomicAdd(&a.tickets[c0], ticket_step(gave_up));
                const bool last = ticket_last(before, pieces);
                if (last) a.tickets[c0] = 0;
                if (last && ticket_complete(before, gave_up)) sm.late[sm.n_late++] = Late{p.q, p.hkv, p.rows, c0, pieces};
            }
        }
        bar_consumers();   // (also: everybody has read the unfinite values)
        if (sm.any_unfinite) {
            for (uint32_t i = tid; i < 3 * D; i += kWarps * 32) (&sm.unfinite[0][0])[i] = 0x7fffffffu;
            bar_consumers();
            if (tid == 0) sm.any_unfinite = 0;
        }
        bar_consumers();   // the shared arrays are free for the next piece
    } while (next_piece(a, walk, p));
    // (the last: every copy into the ring has been waited for, unless a wait ran out)
    if (sm.n_late && !sm.abort_flag) {
        fence_acq_rel_gpu();
        for (uint32_t i = 0; i < sm.n_late; ++i) combine<D, B>(a, sm, sm.late[i]);
    }
    griddep_launch_dependents();
}

template <int D> constexpr size_t few_smem() { return sizeof(FewSmem<D>) + 1024; }

} // namespace

static const struct { void (*k)(const PagedAttnArgs); size_t smem; } kFewKernels[2][3] = {
    {{paged_few_kernel<64, 1>, few_smem<64>()}, {paged_few_kernel<64, 2>, few_smem<64>()}, {paged_few_kernel<64, 4>, few_smem<64>()}},
    {{paged_few_kernel<128, 1>, few_smem<128>()}, {paged_few_kernel<128, 2>, few_smem<128>()}, {paged_few_kernel<128, 4>, few_smem<128>()}}};

cudaError_t paged_few_init(void) {
    for (const auto &row : kFewKernels)
        for (const auto &k : row)
            if (const cudaError_t e = cudaFuncSetAttribute(k.k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem)) return e;
    return cudaSuccess;
}

size_t paged_few_part_bytes(int sms) { return (size_t)4 * sms * kRowsB * (128 + 4) * sizeof(float); }

cudaError_t launch_paged_few(PagedAttnArgs a, const void *k, const void *v, uint32_t head_dim, int sms, cudaStream_t stream) {
    const uint64_t rows = (uint64_t)a.n_pages * a.n_kv << a.page_shift;
    const uint32_t box = std::min(1u << a.page_shift, kTile), grid = 2 * (uint32_t)sms;
    if (grid > kPagedTickets) return cudaErrorInvalidConfiguration;
    if (const cudaError_t e = tensor_map_groups_swz(&a.kmap, k, rows, head_dim, box)) return e;
    if (const cudaError_t e = tensor_map_groups_swz(&a.vmap, v, rows, head_dim, box)) return e;
    const uint64_t most = std::min<uint64_t>((uint64_t)a.max_new * a.group, kRowsB);
    // Fewer blocks of rows at most, fewer registers and instructions. us at 4 x 65000, 32 x 4000 and 1 x 8000 keys: 4 rows 150, 75, 17.4 (as part of
    // 16: 154, 76, 18.4), 8 rows 158, 80, 24.6 (163, 83, 26.2).
    const auto &k_ = kFewKernels[head_dim == 128][most <= 4 ? 0 : most <= 8 ? 1 : 2];
    return launch_kernel(k_.k, dim3(grid), dim3(kThreads), k_.smem, stream, true, a);
}

} // namespace flb
