// Attention over a paged cache, few rows per sequence and KV head: up to 16 rows (token, query head of the group) against tiles
// of 64 keys on mma.sync.
//
// o_r = sum_j exp(s_rj - m_r) v_j / sum_j exp(s_rj - m_r), s_rj = scale q_r . k_j, with the running maximum and sum of an online
// softmax in f32. Bound by the HBM bytes of the keys and values: every tile is read once.
//
// CTA = 4 consumer warps + 1 producer warp, two CTAs per SM. The producer's lanes each copy one page's part of a tile (one TMA box
// of up to 64 rows) into a ring of three stages of 32 KB; warp w takes keys 16 w .. 16 w + 15 of a tile through
// ldmatrix. All tiles lie on one line (sequence, KV head, tile) and every CTA takes an equal piece of it.
//   scores : A = 16 rows of q as (hi, lo) f16 parts, scaled by a power of two per row so that both parts stay normal numbers; B = K
//   softmax: lane (g, t) has rows g and g + 8, keys 2t, 2t + 1 of every 8; row maxima over the 4 lanes of a row
//   context: A = probabilities as (hi, lo) parts: the scores' accumulators have the layout of that operand; B = V (ldmatrix.trans).
//            A tile's product starts from zero and is added in f32 with rounding, since the tensor cores truncate their running sum
//            (1.3e-8 of it per instruction: 1e-5 after 800 tiles).
// A masked value never meets the tensor core as it is, since 0 x NaN is NaN: rows behind the last key are cleared in shared
// memory, and among the keys of the new tokens, which not all rows attend, values that are not finite are taken out there and
// their effect added to the rows that do attend them (see unfinite_of).
#include "common.cuh"
#include "paged.h"

#include <algorithm>

namespace flb {

namespace {

constexpr uint32_t kRowsB = 16, kTile = 64, kStages = 3, kWarps = 4, kThreads = (kWarps + 1) * 32;
constexpr float kShift = 12.f;   // probabilities are 2^(x - m + 12): their lo parts stay normal f16 numbers down to 2^-14 of the largest

template <int D> struct FewSmem {
    static constexpr uint32_t kHalfStage = kTile * D * 2;                 // K or V of a tile
    uint8_t ring[kStages][2 * kHalfStage];                                // 1024-byte aligned
    float o[kWarps][kRowsB][36];                                          // a quarter (half, D = 64) of the warps' contexts
    float m[kWarps][kRowsB], l[kWarps][kRowsB];
    uint32_t unfinite[3][D];                                              // see unfinite_of
    uint64_t full[kStages], empty[kStages];
    uint64_t sum[kThreads / 32];
    uint32_t start_seq, any;
    uint64_t start_off, total;
};

// Values of +inf, -inf and NaN (class 0, 1, 2) among the keys that only part of the rows attend: per class and dimension the
// first such key. A row that attends keys 0 .. lim is affected by those <= lim.
__device__ __forceinline__ float unfinite_of(const uint32_t *u, uint32_t dims, uint32_t d, int32_t lim) {
    const int32_t p = (int32_t)u[d], n = (int32_t)u[dims + d], x = (int32_t)u[2 * dims + d];   // (0x7fffffff: none)
    if (x <= lim || (p <= lim && n <= lim)) return __int_as_float(0x7fffffff);
    return p <= lim ? INFINITY : n <= lim ? -INFINITY : 0.f;
}

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
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// (a, b) as two f16 pairs, hi + lo
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = half2_bits(a - f.x, b - f.y);
}
__device__ __forceinline__ void bar_consumers() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t *bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }

// Rows of a sequence over one KV head, 0 where it is the other kernel's; its tiles: at least one, so that somebody writes its rows.
__device__ __forceinline__ uint32_t rows_of(const PagedAttnArgs &a, const PagedSeq &q) { return q.n * a.group > a.few_rows ? 0u : q.n * a.group; }
__device__ __forceinline__ uint32_t tiles_of(const PagedSeq &q) { return max(1u, ((uint32_t)max(0, q.past + (int32_t)q.n) + kTile - 1) / kTile); }
__device__ __forceinline__ uint64_t units_of(const PagedAttnArgs &a, const PagedSeq &q) { return rows_of(a, q) ? (uint64_t)tiles_of(q) * a.n_kv : 0u; }

// The pieces of a CTA's share: consecutive tiles of one sequence over one KV head.
struct Piece {
    PagedSeq q;
    uint32_t seq, hkv, rows, tiles, t0, t1;        // tiles t0 .. t1 - 1 of `tiles`
    int32_t keys;
    uint64_t base;                                 // unit of its tile 0
};
struct Walk {
    uint64_t pos, hi, seq_base;   // seq_base: first unit of sequence `seq`
    uint32_t seq;
    bool fresh;
};
// The next piece; p keeps the state between calls.
__device__ __forceinline__ bool next_piece(const PagedAttnArgs &a, Walk &w, Piece &p) {
    if (w.pos >= w.hi) return false;
    bool bad;
    if (w.fresh) {
        w.fresh = false;
        p.seq = w.seq;
        p.q = paged_seq(a, p.seq, bad);
        p.rows = rows_of(a, p.q);
        p.tiles = tiles_of(p.q);
        p.hkv = (uint32_t)((w.pos - w.seq_base) / p.tiles);
        p.base = w.seq_base + (uint64_t)p.hkv * p.tiles;
    } else {
        p.base += p.tiles;
        if (++p.hkv == a.n_kv) {
            p.hkv = 0;
            do { p.q = paged_seq(a, ++p.seq, bad); } while ((p.rows = rows_of(a, p.q)) == 0);
            p.tiles = tiles_of(p.q);
        }
    }
    p.keys = max(0, p.q.past + (int32_t)p.q.n);
    p.t0 = (uint32_t)(w.pos - p.base);
    p.t1 = (uint32_t)min((uint64_t)p.tiles, w.hi - p.base);
    w.pos += p.t1 - p.t0;
    return true;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2) paged_few_kernel(const __grid_constant__ PagedAttnArgs a) {
    extern __shared__ uint8_t smem_dyn[];
    FewSmem<D> &sm = *reinterpret_cast<FewSmem<D> *>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
    constexpr uint32_t kKV = FewSmem<D>::kHalfStage, kGroupBytes = 8 * D * 2;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, t = lane & 3u;
    if (tid == 0) {
        for (uint32_t s = 0; s < kStages; ++s) { mbar_init(&sm.full[s], 1); mbar_init(&sm.empty[s], kWarps); }
        fence_barrier_init();
    }
    for (uint32_t i = tid; i < 3 * D; i += kThreads) (&sm.unfinite[0][0])[i] = 0x7fffffffu;
    griddep_wait();

    // ---- this CTA's share of the line ----
    {
        const uint32_t per = (a.n_seq + kThreads - 1) / kThreads, s0 = min(tid * per, a.n_seq), s1 = min(s0 + per, a.n_seq);
        uint64_t mine = 0;
        bool bad = false, any_bad = false;
        for (uint32_t s = s0; s < s1; ++s) {
            mine += units_of(a, paged_seq(a, s, bad));
            any_bad |= bad;
        }
        if (any_bad && blockIdx.x == 0) atomicCAS(a.status, ST_OK, ST_PAGED_ARGS);
        uint64_t x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t u = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += u;
        }
        if (lane == 31) sm.sum[warp] = x;
        __syncthreads();
        uint64_t total = 0;
        for (uint32_t w = 0; w < kThreads / 32; ++w) {
            if (w < warp) x += sm.sum[w];
            total += sm.sum[w];
        }
        x -= mine;
        const uint32_t ctas = (uint32_t)min((uint64_t)gridDim.x, total);
        if (blockIdx.x >= ctas) return;   // (no share is empty: the CTAs of a block's records are consecutive)
        const uint64_t lo = share_of(total, ctas, blockIdx.x);
        if (tid == 0) sm.total = total;
        if (lo >= x && lo < x + mine) {
            uint32_t s = s0;
            for (;; ++s) {
                const uint64_t u = units_of(a, paged_seq(a, s, bad));
                if (lo < x + u) break;
                x += u;
            }
            sm.start_seq = s;
            sm.start_off = x;
        }
        __syncthreads();
    }
    const uint64_t total = sm.total;
    const uint32_t ctas = (uint32_t)min((uint64_t)gridDim.x, total);
    Walk walk{share_of(total, ctas, blockIdx.x), share_of(total, ctas, blockIdx.x + 1), sm.start_off, sm.start_seq, true};
    Piece p;
    uint32_t stage = 0, parity = 0;   // of the ring

    if (warp == kWarps) {
        // ---- producer ----
        const uint32_t box = min(1u << a.page_shift, kTile), boxes = kTile / box, bytes = box * D * 2;
        const uint32_t page_groups = (1u << a.page_shift) >> 3, outside = a.n_pages * a.n_kv * page_groups;
        while (next_piece(a, walk, p)) {
            const int32_t *row = a.table + (uint64_t)p.seq * a.max_blocks;
            auto page_at = [&](uint32_t tile) -> int32_t {   // the page that this lane's part of the tile lies on; -1: behind the last key
                const uint32_t key = tile * kTile + lane * box;
                return lane < boxes && key < (uint32_t)p.keys ? row[key >> a.page_shift] : -1;
            };
            int32_t page = page_at(p.t0);
            for (uint32_t tile = p.t0; tile < p.t1; ++tile) {
                const uint32_t key = tile * kTile + lane * box;
                uint32_t at = outside;   // copies from there bring zeros
                if (lane < boxes && key < (uint32_t)p.keys) {
                    if ((uint32_t)page < a.n_pages)
                        at = ((uint32_t)page * a.n_kv + p.hkv) * page_groups + ((key & ((1u << a.page_shift) - 1u)) >> 3);
                    else
                        atomicCAS(a.status, ST_OK, ST_PAGED_PAGE);
                }
                if (tile + 1 < p.t1) page = page_at(tile + 1);
                if (!mbar_wait_bounded(&sm.empty[stage], parity ^ 1u, a.status)) return;
                if (lane == 0) mbar_arrive_expect_tx(&sm.full[stage], 2 * kKV);
                __syncwarp();
                if (lane < boxes) {
                    const uint32_t dst = smem_u32(sm.ring[stage]) + lane * bytes, bar = smem_u32(&sm.full[stage]);
                    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3}], [%4];" ::"r"(dst),
                                 "l"(&a.kmap), "r"(0u), "r"(at), "r"(bar) : "memory");
                    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3}], [%4];" ::"r"(dst + kKV),
                                 "l"(&a.vmap), "r"(0u), "r"(at), "r"(bar) : "memory");
                }
                if (++stage == kStages) { stage = 0; parity ^= 1u; }
            }
        }
        griddep_launch_dependents();
        return;
    }

    // ---- consumers ----
    bool first = true;
    while (next_piece(a, walk, p)) {
        // q: rows g and g + 8, dimensions 2t, 2t + 1 of every 8
        uint32_t qh[D / 16][4], ql[D / 16][4];
        float f[2];        // score -> exponent of 2, per row
        int32_t lim[2];    // last key of a row
        {
            float x[2][D / 4];
            bool there[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint32_t row = g + 8 * r, tok = row / a.group, head = p.hkv * a.group + row - tok * a.group;
                there[r] = row < p.rows;
                lim[r] = there[r] ? p.q.past + (int32_t)tok : -1;
                const uint64_t src = there[r] ? (p.q.first + tok) * a.q_stride + (uint64_t)head * D : 0;
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    float2 v = make_float2(0.f, 0.f);
                    if (there[r]) {
                        if (a.half) v = __half22float2(*reinterpret_cast<const __half2 *>((const __half *)a.q + src + 8 * j + 2 * t));
                        else v = *reinterpret_cast<const float2 *>((const float *)a.q + src + 8 * j + 2 * t);
                    }
                    x[r][2 * j] = v.x; x[r][2 * j + 1] = v.y;
                }
                float top = 0.f;
#pragma unroll
                for (int j = 0; j < D / 4; ++j) top = fmaxf(top, fabsf(x[r][j]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // a power of two brings the row's largest value to [2^11, 2^12)
                const int e = min(100, max(-100, 138 - (int)(__float_as_uint(top) >> 23)));
                const float up = __uint_as_float((uint32_t)(e + 127) << 23);
                f[r] = a.scale * 1.44269504088896341f * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                for (int j = 0; j < D / 4; ++j) x[r][j] *= up;
            }
#pragma unroll
            for (int kb = 0; kb < D / 16; ++kb)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    split2(x[r][4 * kb], x[r][4 * kb + 1], qh[kb][r], ql[kb][r]);
                    split2(x[r][4 * kb + 2], x[r][4 * kb + 3], qh[kb][2 + r], ql[kb][2 + r]);
                }
        }
        const int32_t lim_first = p.q.past;   // last key that all rows attend
        float o[D / 8][4];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        for (uint32_t tile = p.t0; tile < p.t1; ++tile) {
            if (!mbar_wait_bounded(&sm.full[stage], parity, a.status)) return;
            const int32_t k0 = (int32_t)(tile * kTile + warp * 16);
            if (k0 < p.keys) {
                const uint32_t kb_s = smem_u32(sm.ring[stage]) + warp * 2 * kGroupBytes, vb_s = kb_s + kKV;
                if (k0 + 16 > lim_first + 1 || k0 + 16 > p.keys) {
                    uint8_t *vrow = sm.ring[stage] + kKV + warp * 2 * kGroupBytes;
                    for (uint32_t i = lane; i < 16 * D / 8; i += 32) {
                        const uint32_t r = i / (D / 8), c = i % (D / 8);
                        const int32_t key = k0 + (int32_t)r;
                        uint4 *at = reinterpret_cast<uint4 *>(vrow + (r >> 3) * kGroupBytes + (c >> 3) * 1024 + (r & 7u) * 128 + (((c ^ r) & 7u) << 4));
                        if (key >= p.keys) {
                            *at = make_uint4(0, 0, 0, 0);
                        } else if (key > lim_first) {
                            uint4 v = *at;
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                            uint32_t z = 0;
#pragma unroll
                            for (int j = 0; j < 4; ++j) z |= (w[j] & 0x7C007C00u) + 0x04000400u;
                            if (z & 0x80008000u) {   // an exponent of all ones
                                __half *h = reinterpret_cast<__half *>(at);
                                for (uint32_t j = 0; j < 8; ++j) {
                                    const uint16_t b = __half_as_ushort(h[j]);
                                    if ((b & 0x7C00u) == 0x7C00u) {
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
                // ---- scores ----
                float sh[2][4], sl[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sh[n][i] = sl[n][i] = 0.f;
                const uint32_t mi = lane >> 3, r8 = lane & 7u;
#pragma unroll
                for (int kb = 0; kb < D / 16; ++kb) {
                    uint32_t b[4];
                    ldsm4(kb_s + (mi >> 1) * kGroupBytes + (kb >> 2) * 1024 + r8 * 128 + (((2 * (kb & 3) + (mi & 1u)) ^ r8) << 4), b);
                    mma(sh[0], qh[kb], b[0], b[1]);
                    mma(sh[1], qh[kb], b[2], b[3]);
                    mma(sl[0], ql[kb], b[0], b[1]);
                    mma(sl[1], ql[kb], b[2], b[3]);
                }
                // ---- softmax: value 2 r + i of n: row g + 8 r, key 8 n + 2 t + i ----
                float al[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float x[4];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float s = sh[n][2 * r + i] + sl[n][2 * r + i];
                            x[2 * n + i] = k0 + 8 * n + (int32_t)(2 * t) + i <= lim[r] ? s : -INFINITY;
                        }
                    float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float mn = fmaxf(m[r], top * f[r]), ref = (mn == -INFINITY ? 0.f : mn) - kShift;
                    al[r] = exp2_fast(m[r] - kShift - ref);
                    m[r] = mn;
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float e = exp2_fast(fmaf(x[j], f[r], -ref));
                        sum += e;
                        sh[j >> 1][2 * r + (j & 1)] = e;
                    }
                    l[r] = fmaf(l[r], al[r], sum);
                }
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int r = 0; r < 2; ++r) split2(sh[n][2 * r], sh[n][2 * r + 1], ph[2 * n + r], pl[2 * n + r]);
                // ---- context ----
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    uint32_t b[4];
                    ldsm4t(vb_s + (mi & 1u) * kGroupBytes + (j >> 2) * 1024 + r8 * 128 + (((2 * (j & 3) + (mi >> 1)) ^ r8) << 4), b);
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                        mma(d, pl, b[2 * n], b[2 * n + 1]);
                        mma(d, ph, b[2 * n], b[2 * n + 1]);
                        float (&w)[4] = o[2 * j + n];
                        w[0] = fmaf(w[0], al[0], d[0]); w[1] = fmaf(w[1], al[0], d[1]);
                        w[2] = fmaf(w[2], al[1], d[2]); w[3] = fmaf(w[3], al[1], d[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) arrive(&sm.empty[stage]);
            if (++stage == kStages) { stage = 0; parity ^= 1u; }
        }

        // ---- the warps' sums, a part of the dimensions at a time ----
        const uint32_t c0 = owner_of(total, ctas, p.base), c1 = owner_of(total, ctas, p.base + p.tiles - 1), pieces = c1 - c0 + 1;
        const bool whole = pieces == 1;
        float *rec = a.part + (uint64_t)(blockIdx.x * 2 + (first ? 0 : 1)) * kRowsB * (D + 4);
        first = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t == 0) { sm.m[warp][g + 8 * r] = m[r]; sm.l[warp][g + 8 * r] = l[r]; }
        }
        bar_consumers();
        float wgt[2];   // this warp's weight, rows g, g + 8
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) top = fmaxf(top, sm.m[w][g + 8 * r]);
            wgt[r] = m[r] == -INFINITY && top != -INFINITY ? 0.f : exp2_fast(top == -INFINITY ? 0.f : m[r] - top);
        }
        const uint32_t row = tid >> 3, c4 = (tid & 7u) * 4;   // the thread's row and 4 of a part's 32 dimensions
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) top = fmaxf(top, sm.m[w][row]);
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) sum = fmaf(sm.l[w][row], sm.m[w][row] == -INFINITY && top != -INFINITY ? 0.f : exp2_fast(top == -INFINITY ? 0.f : sm.m[w][row] - top), sum);
        const uint32_t tok = row / a.group, head = p.hkv * a.group + row - tok * a.group;
        const int32_t row_lim = p.q.past + (int32_t)tok;
        const uint64_t dst = (p.q.first + tok) * a.out_stride + (uint64_t)head * D;
        auto put = [&](uint64_t to, const float4 &v) {
            if (a.half) *reinterpret_cast<uint2 *>((__half *)a.out + to) = make_uint2(half2_bits(v.x, v.y), half2_bits(v.z, v.w));
            else *reinterpret_cast<float4 *>((float *)a.out + to) = v;
        };
        auto put_lse = [&](uint32_t tk, uint32_t hd, float mx, float s) {
            a.lse[(uint64_t)(p.q.first + tk) * a.n_kv * a.group + hd] = make_float2(mx * 0.693147180559945309f, s * 0.000244140625f);   // 2^-kShift
        };
        for (uint32_t part = 0; part < D / 32; ++part) {
            if (part) bar_consumers();
#pragma unroll
            for (int j = 0; j < D / 8; ++j)
                if ((uint32_t)j / 4 == part)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        *reinterpret_cast<float2 *>(&sm.o[warp][g + 8 * r][(j & 3) * 8 + 2 * t]) = make_float2(o[j][2 * r] * wgt[r], o[j][2 * r + 1] * wgt[r]);
            bar_consumers();
            if (row < p.rows) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) {
                    const float4 u = *reinterpret_cast<const float4 *>(&sm.o[w][row][c4]);
                    v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
                }
                const uint32_t d = part * 32 + c4;
                v.x += unfinite_of(&sm.unfinite[0][0], D, d, row_lim); v.y += unfinite_of(&sm.unfinite[0][0], D, d + 1, row_lim);
                v.z += unfinite_of(&sm.unfinite[0][0], D, d + 2, row_lim); v.w += unfinite_of(&sm.unfinite[0][0], D, d + 3, row_lim);
                if (whole) {
                    const float inv = row_lim < 0 ? 0.f : 1.f / sum;
                    put(dst + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                } else {
                    __stcg(reinterpret_cast<float4 *>(rec + row * (D + 4) + d), v);
                }
            }
        }
        if (row < p.rows && c4 == 0) {
            if (whole) { if (a.lse) put_lse(tok, head, top, sum); }
            else __stcg(reinterpret_cast<float4 *>(rec + row * (D + 4) + D), make_float4(top, sum, 0.f, 0.f));
        }
        if (!whole) {
            __threadfence();
            bar_consumers();
            if (tid == 0) sm.any = atomicAdd(&a.tickets[c0], 1u) == pieces - 1 ? 1u : 0u;
        }
        bar_consumers();   // (also: everybody has read the unfinite values)
        for (uint32_t i = tid; i < 3 * D; i += kWarps * 32) (&sm.unfinite[0][0])[i] = 0x7fffffffu;
        if (!whole && sm.any) {
            __threadfence();
            // the records in order: of CTA c0 the piece at its end, of the others the one at their start
            const bool c0_first = p.base <= share_of(total, ctas, c0);
            auto record = [&](uint32_t i, uint32_t rw) { return a.part + ((uint64_t)((c0 + i) * 2 + (i || c0_first ? 0 : 1)) * kRowsB + rw) * (D + 4); };
            for (uint32_t i = tid; i < p.rows * (D / 4); i += kWarps * 32) {
                const uint32_t rw = i / (D / 4), d = i % (D / 4) * 4;
                float mx = -INFINITY;
#pragma unroll 8
                for (uint32_t k = 0; k < pieces; ++k) mx = fmaxf(mx, __ldcg(record(k, rw) + D));
                float s = 0.f;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                for (uint32_t k = 0; k < pieces; ++k) {
                    const float *rc = record(k, rw);
                    const float2 ml = __ldcg(reinterpret_cast<const float2 *>(rc + D));
                    const float4 u = __ldcg(reinterpret_cast<const float4 *>(rc + d));
                    const float w = ml.x == -INFINITY && mx != -INFINITY ? 0.f : exp2_fast(mx == -INFINITY ? 0.f : ml.x - mx);
                    s = fmaf(ml.y, w, s);
                    v.x = fmaf(u.x, w, v.x); v.y = fmaf(u.y, w, v.y); v.z = fmaf(u.z, w, v.z); v.w = fmaf(u.w, w, v.w);
                }
                const uint32_t tk = rw / a.group, hd = p.hkv * a.group + rw - tk * a.group;
                const float inv = p.q.past + (int32_t)tk < 0 ? 0.f : 1.f / s;
                put((p.q.first + tk) * a.out_stride + (uint64_t)hd * D + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                if (a.lse && d == 0) put_lse(tk, hd, mx, s);
            }
            if (tid == 0) a.tickets[c0] = 0;
        }
        bar_consumers();   // the shared arrays are free for the next piece
    }
    griddep_launch_dependents();
}

template <int D> constexpr size_t few_smem() { return sizeof(FewSmem<D>) + 1024; }

} // namespace

cudaError_t paged_few_init(void) {
    if (const cudaError_t e = cudaFuncSetAttribute(paged_few_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)few_smem<64>())) return e;
    return cudaFuncSetAttribute(paged_few_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)few_smem<128>());
}

size_t paged_few_part_bytes(int sms) { return (size_t)4 * sms * kRowsB * (128 + 4) * sizeof(float); }

cudaError_t launch_paged_few(PagedAttnArgs a, const void *k, const void *v, uint32_t head_dim, int sms, cudaStream_t stream) {
    const uint64_t rows = (uint64_t)a.n_pages * a.n_kv << a.page_shift;
    const uint32_t box = std::min(1u << a.page_shift, kTile), grid = 2 * (uint32_t)sms;
    if (grid > kPagedTickets) return cudaErrorInvalidConfiguration;
    if (const cudaError_t e = tensor_map_groups_swz(&a.kmap, k, rows, head_dim, box)) return e;
    if (const cudaError_t e = tensor_map_groups_swz(&a.vmap, v, rows, head_dim, box)) return e;
    return head_dim == 128 ? launch_kernel(paged_few_kernel<128>, dim3(grid), dim3(kThreads), few_smem<128>(), stream, true, a)
                           : launch_kernel(paged_few_kernel<64>, dim3(grid), dim3(kThreads), few_smem<64>(), stream, true, a);
}

} // namespace flb
