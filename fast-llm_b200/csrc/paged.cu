// Paged KV cache: the C ABI of its three operators (include/fl_b200.h), the plan of a step (block tables, slot maps and positions
// from the requests' lengths) and the append of a ragged batch of tokens. Attention over pages: attn_paged.cu.
// The reference has neither pages nor several sequences; the operators these extend are fl_op_rope_ds2, fl_op_kv_append and
// fl_op_attn_head (src/runtime/decode_params.h:124-232).
#include "capi_internal.h"
#include "paged.h"

#include <algorithm>
#include <cmath>

namespace flb {

namespace {

// ---- plan -----------------------------------------------------------------------------------------------------------
// Three prefix sums over the sequences (new tokens, pages taken, pages given back), formed by every CTA for itself in shared
// memory, make all outputs independent of one another: token i finds its sequence by a search in the first; a page taken is the
// k-th from the top of the stack, that is an entry of the old stack or, past its end, a page given back, found by a search in
// the third. Nothing that a CTA reads is written by another one: new table entries lie behind the old ones, returned pages behind
// the old stack, and kv_len and the new count, which may overwrite inputs, are the last CTA's to write.
constexpr uint32_t kPlanThreads = 512;

struct PlanArgs {
    const int32_t *held, *past, *fresh;
    int32_t *table, *free_list;
    const int32_t *free_in;
    int32_t *free_out, *q_start, *kv_len, *pos, *slot;
    uint32_t *ticket, *status;
    uint32_t n_seq, page_shift, max_blocks, n_pages, max_tokens;
};

__device__ __forceinline__ uint64_t warp_scan(uint64_t v, uint32_t lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += u;
    }
    return v;
}
// The last index whose prefix is <= v, of n + 1 ascending ones (the first is 0, v below the last): the entry that holds v.
__device__ __forceinline__ uint32_t find_in(const uint32_t *prefix, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;   // prefix[lo] <= v < prefix[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (prefix[mid] <= v) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanArgs a) {
    extern __shared__ uint32_t plan_smem[];
    uint32_t *tok = plan_smem, *take = tok + a.n_seq + 1, *give = take + a.n_seq + 1;
    __shared__ uint64_t wsum[3][kPlanThreads / 32];
    __shared__ uint32_t last;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    griddep_launch_dependents();
    griddep_wait();
    const uint32_t round_up = (1u << a.page_shift) - 1u;
    auto pages_of = [&](uint32_t n) { return (n + round_up) >> a.page_shift; };
    const int64_t most = (int64_t)a.max_blocks << a.page_shift;   // (below 2^31)
    bool bad = false;
    uint64_t run[3] = {0, 0, 0};
    for (uint32_t s0 = 0; s0 < a.n_seq; s0 += kPlanThreads) {
        const uint32_t s = s0 + tid;
        uint64_t v[3] = {0, 0, 0};
        if (s < a.n_seq) {
            const int64_t h = a.held[s], p = a.past[s], n = a.fresh[s];
            if (h < 0 || p < 0 || n < 0 || p > h || h > most || p + n > most) {
                bad = true;
            } else {
                const uint32_t have = pages_of((uint32_t)h), need = pages_of((uint32_t)(p + n));
                v[0] = (uint64_t)n;
                v[1] = need > have ? need - have : 0;
                v[2] = have > need ? have - need : 0;
            }
        }
        uint64_t x[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            x[k] = warp_scan(v[k], lane);
            if (lane == 31) wsum[k][warp] = x[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            uint64_t before = 0, all = 0;
#pragma unroll
            for (uint32_t w = 0; w < kPlanThreads / 32; ++w) {
                const uint64_t t = wsum[k][w];
                if (w < warp) before += t;
                all += t;
            }
            x[k] += run[k] + before - v[k];   // exclusive
            run[k] += all;
        }
        if (s < a.n_seq) { tok[s] = (uint32_t)x[0]; take[s] = (uint32_t)x[1]; give[s] = (uint32_t)x[2]; }
        __syncthreads();
    }
    const int64_t have_free = a.free_in[0];
    bad = __syncthreads_or(bad) || have_free < 0 || (uint64_t)have_free + run[2] > a.n_pages;
    const bool full = run[0] > a.max_tokens || run[1] > (uint64_t)have_free + run[2];
    const bool ok = !bad && !full;
    const uint32_t n_tok = ok ? (uint32_t)run[0] : 0u, F = (uint32_t)have_free, R = (uint32_t)run[2], T = (uint32_t)run[1];
    if (tid == 0) { tok[a.n_seq] = (uint32_t)run[0]; take[a.n_seq] = T; give[a.n_seq] = R; }
    __syncthreads();

    const uint32_t gthread = blockIdx.x * kPlanThreads + tid, threads = gridDim.x * kPlanThreads;
    if (ok) {
        // the k-th page taken (in order of sequence and block) is the k-th from the top of the stack with the returned pages on it
        auto popped = [&](uint32_t k) -> int32_t {
            const uint32_t x = F + R - 1u - k;
            if (x < F) return a.free_list[x];
            const uint32_t g = x - F, s = find_in(give, a.n_seq, g);
            return a.table[(uint64_t)s * a.max_blocks + pages_of((uint32_t)(a.past[s] + a.fresh[s])) + (g - give[s])];
        };
        // pages taken: table entries; pages given back and not taken again: onto the stack
        for (uint32_t k = gthread; k < T; k += threads) {
            const uint32_t s = find_in(take, a.n_seq, k);
            a.table[(uint64_t)s * a.max_blocks + pages_of((uint32_t)a.held[s]) + (k - take[s])] = popped(k);
        }
        for (uint32_t g = gthread; g + T < R; g += threads) {
            const uint32_t s = find_in(give, a.n_seq, g);
            a.free_list[F + g] = a.table[(uint64_t)s * a.max_blocks + pages_of((uint32_t)(a.past[s] + a.fresh[s])) + (g - give[s])];
        }
        for (uint32_t i = gthread; i < n_tok; i += threads) {
            const uint32_t s = find_in(tok, a.n_seq, i), p = (uint32_t)a.past[s] + (i - tok[s]), j = p >> a.page_shift,
                           have = pages_of((uint32_t)a.held[s]);
            const int32_t page = j < have ? a.table[(uint64_t)s * a.max_blocks + j] : popped(take[s] + j - have);
            // (a page whose slots 31 bits do not hold would come out as another page's)
            const bool there = (uint32_t)page <= 0x7fffffffu >> a.page_shift;
            if (!there) atomicCAS(a.status, ST_OK, ST_PAGED_PAGE);
            a.pos[i] = (int32_t)p;
            a.slot[i] = there ? (int32_t)(((uint32_t)page << a.page_shift) | (p & round_up)) : -1;
        }
    }
    for (uint32_t i = n_tok + gthread; i < a.max_tokens; i += threads) { a.pos[i] = -1; a.slot[i] = -1; }
    for (uint32_t s = gthread; s <= a.n_seq; s += threads) a.q_start[s] = ok ? (int32_t)tok[s] : 0;
    if (gridDim.x > 1) {
        __threadfence();
        __syncthreads();
        if (tid == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1 ? 1u : 0u;
        __syncthreads();
        if (!last) return;
        if (tid == 0) *a.ticket = 0;
        __threadfence();
    } else {
        __syncthreads();
    }
    if (ok)
        for (uint32_t s = tid; s < a.n_seq; s += kPlanThreads) a.kv_len[s] = a.past[s] + a.fresh[s];
    if (tid == 0) {
        a.free_out[0] = ok ? (int32_t)(F + R - T) : (int32_t)have_free;
        if (!ok) atomicCAS(a.status, ST_OK, bad ? ST_PAGED_ARGS : ST_PAGED_FULL);
    }
}

// ---- append ---------------------------------------------------------------------------------------------------------
// Bound by HBM bytes. A CTA has one token (8192 tokens, 8B shape, f32: 66 us, four of them 69, eight 73), few tokens several CTAs each: the angles' sines and
// cosines once in shared memory, then every thread 16 bytes of one head at a time, the next ones' load in flight. The angle pos *
// base^(-2i/n) is formed in turns in 64 bits and reduced before it is rounded: in 32 bits a position of 120000 is 0.004 radians off.
constexpr uint32_t kAppThreads = 256;

struct AppendArgs {
    const void *q, *k, *v;
    void *q_out;
    __half *kc, *vc;
    const int32_t *pos, *slot;
    uint32_t *status;
    uint64_t q_stride, kv_stride, q_out_stride;
    uint32_t n_q, n_kv, dim_shift, n_rot, page_shift, n_pages;
    double turns[64];               // base^(-2i/n_rot) / 2 pi
};

template <typename T> struct AppVec;
template <> struct AppVec<float> {
    static constexpr uint32_t N = 4;
    static __device__ __forceinline__ void load(const float *p, float (&x)[N]) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
    static __device__ __forceinline__ void store(float *p, const float (&x)[N]) { *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]); }
};
template <> struct AppVec<__half> {
    static constexpr uint32_t N = 8;
    static __device__ __forceinline__ void load(const __half *p, float (&x)[N]) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void store(__half *p, const float (&x)[N]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <typename T>
__global__ void __launch_bounds__(kAppThreads) paged_append_kernel(const __grid_constant__ AppendArgs a) {
    __shared__ float2 cs[64];   // cosine, sine per pair
    constexpr uint32_t N = AppVec<T>::N;
    const uint32_t tid = threadIdx.x, tok = blockIdx.x, half = a.n_rot / 2;
    const uint32_t vec_shift = a.dim_shift - (N == 4 ? 2u : 3u), n_vec = (a.n_q + 2 * a.n_kv) << vec_shift, step = gridDim.y * kAppThreads;
    griddep_launch_dependents();
    griddep_wait();
    const int32_t pos = a.pos[tok], slot = a.slot[tok];
    if (pos < 0) return;   // a row behind the last token
    const uint32_t page = (uint32_t)slot >> a.page_shift;
    const bool stored = slot >= 0 && page < a.n_pages;
    if (slot >= 0 && !stored && tid == 0) atomicCAS(a.status, ST_OK, ST_PAGED_PAGE);
    // piece i: its head, its dimension, where it comes from
    auto head_of = [&](uint32_t i) { return i >> vec_shift; };
    auto dim_of = [&](uint32_t i) { return (i & ((1u << vec_shift) - 1u)) * N; };
    auto wanted = [&](uint32_t i) { return i < n_vec && (stored || head_of(i) < a.n_q); };
    auto load = [&](uint32_t i, float (&x)[N]) {
        const uint32_t h = head_of(i);
        const T *src = h < a.n_q ? (const T *)a.q + tok * a.q_stride + ((uint64_t)h << a.dim_shift)
                                 : (const T *)(h < a.n_q + a.n_kv ? a.k : a.v) + tok * a.kv_stride + ((uint64_t)(h - a.n_q - (h < a.n_q + a.n_kv ? 0u : a.n_kv)) << a.dim_shift);
        AppVec<T>::load(src + dim_of(i), x);
    };
    float x[N];
    uint32_t i = blockIdx.y * kAppThreads + tid;
    if (wanted(i)) load(i, x);   // (in flight while the angles are formed)
    for (uint32_t p = tid; p < half; p += kAppThreads) {
        const double turn = (double)pos * a.turns[p];
        float s, c;
        sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
        cs[p] = make_float2(c, s);
    }
    __syncthreads();
    for (; i < n_vec; i += step) {
        if (wanted(i)) {
            const uint32_t h = head_of(i), d = dim_of(i);
            const bool is_q = h < a.n_q, is_v = h >= a.n_q + a.n_kv;
            if (!is_v && d < a.n_rot) {
#pragma unroll
                for (uint32_t j = 0; j < N; j += 2)
                    if (d + j < a.n_rot) {
                        const float2 w = cs[(d + j) / 2];
                        const float x0 = x[j], x1 = x[j + 1];
                        x[j] = fmaf(x0, w.x, -(x1 * w.y));
                        x[j + 1] = fmaf(x0, w.y, x1 * w.x);
                    }
            }
            if (is_q) {
                AppVec<T>::store((T *)a.q_out + tok * a.q_out_stride + ((uint64_t)h << a.dim_shift) + d, x);
            } else {
                const uint64_t row = (((uint64_t)page * a.n_kv + h - a.n_q - (is_v ? a.n_kv : 0u)) << a.page_shift) + ((uint32_t)slot & ((1u << a.page_shift) - 1u));
                __half *dst = (is_v ? a.vc : a.kc) + (row << a.dim_shift) + d;
                uint32_t w[N / 2];
#pragma unroll
                for (uint32_t j = 0; j < N / 2; ++j) {
                    const __half2 y = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t *>(&y);
                }
                if constexpr (N == 4) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        if (wanted(i + step)) load(i + step, x);
    }
}

// Makes the context's device current for the calls of one entry point.
struct OnDevice {
    int before = -1;
    cudaError_t err;
    explicit OnDevice(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
        else before = -1;
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};

bool aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int page_shift_of(uint32_t page_size) {
    for (int s = 4; s <= 8; ++s)
        if (page_size == 1u << s) return s;
    return -1;
}

int check_cache(const char *who, const fl_b200_paged_cache *c, int act) {
    if (!c || !c->k_dev || !c->v_dev) return set_err(FL_B200_ERR_ARG, "%s: null cache", who);
    if (c->head_dim != 64 && c->head_dim != 128) return set_err(FL_B200_ERR_ARG, "%s: head_dim %u (64 and 128 are built)", who, c->head_dim);
    if (page_shift_of(c->page_size) < 0) return set_err(FL_B200_ERR_ARG, "%s: page_size %u (16, 32, 64, 128 or 256)", who, c->page_size);
    if (c->n_kv_head == 0 || c->n_kv_head > 1024) return set_err(FL_B200_ERR_ARG, "%s: %u KV heads", who, c->n_kv_head);
    if (c->n_pages == 0 || (uint64_t)c->n_pages * c->n_kv_head * c->page_size >= (1ull << 31))
        return set_err(FL_B200_ERR_ARG, "%s: %u pages (1 to 2^31 - 1 rows of all KV heads)", who, c->n_pages);
    if (!aligned(c->k_dev, 16) || !aligned(c->v_dev, 16)) return set_err(FL_B200_ERR_ARG, "%s: pools must be 16-byte aligned", who);
    if (act != FL_B200_ACT_F32 && act != FL_B200_ACT_F16) return set_err(FL_B200_ERR_ARG, "%s: activation type %d", who, act);
    return FL_B200_OK;
}

// Rows of n_head heads: their stride holds them and keeps 16-byte pieces aligned.
int check_rows(const char *who, const char *what, const void *p, uint32_t n_head, uint32_t dim, uint32_t stride, int act) {
    if (!p) return set_err(FL_B200_ERR_ARG, "%s: %s is null", who, what);
    if (!aligned(p, 16) || stride % (act == FL_B200_ACT_F16 ? 8 : 4))
        return set_err(FL_B200_ERR_ARG, "%s: %s and its rows must be 16-byte aligned", who, what);
    if (stride < (uint64_t)n_head * dim) return set_err(FL_B200_ERR_ARG, "%s: stride %u of %s is less than a row", who, stride, what);
    return FL_B200_OK;
}

} // namespace

cudaError_t paged_init(void) {
    if (const cudaError_t e = cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(3 * (kPagedMaxSeq + 1) * 4))) return e;
    if (const cudaError_t e = paged_few_init()) return e;
    return paged_tm_init();
}

} // namespace flb

using namespace flb;

extern "C" {

int fl_b200_paged_plan(fl_b200_ctx *c, const int32_t *held, const int32_t *past, const int32_t *fresh, uint32_t n_seq,
                       uint32_t page_size, int32_t *table, uint32_t max_blocks, int32_t *free_list, uint32_t n_pages,
                       const int32_t *free_in, int32_t *free_out, int32_t *q_start, int32_t *kv_len, int32_t *pos, int32_t *slot,
                       uint32_t max_tokens) {
    if (!c) return set_err(FL_B200_ERR_ARG, "paged_plan: null context");
    if (!held || !past || !fresh || !table || !free_list || !free_in || !free_out || !q_start || !kv_len || (max_tokens && (!pos || !slot)))
        return set_err(FL_B200_ERR_ARG, "paged_plan: null pointer");
    if (n_seq == 0 || n_seq > kPagedMaxSeq) return set_err(FL_B200_ERR_ARG, "paged_plan: %u sequences (1 to %u)", n_seq, kPagedMaxSeq);
    const int shift = page_shift_of(page_size);
    if (shift < 0) return set_err(FL_B200_ERR_ARG, "paged_plan: page_size %u (16, 32, 64, 128 or 256)", page_size);
    if (max_blocks == 0 || ((uint64_t)max_blocks << shift) >= (1ull << 31)) return set_err(FL_B200_ERR_ARG, "paged_plan: %u blocks a sequence", max_blocks);
    if (n_pages == 0 || ((uint64_t)n_pages << shift) >= (1ull << 31)) return set_err(FL_B200_ERR_ARG, "paged_plan: %u pages", n_pages);
    if (max_tokens >= (1u << 31)) return set_err(FL_B200_ERR_ARG, "paged_plan: %u tokens", max_tokens);
    for (const void *p : {(const void *)held, (const void *)past, (const void *)fresh, (const void *)table, (const void *)free_list, (const void *)free_in,
                          (const void *)free_out, (const void *)q_start, (const void *)kv_len, (const void *)pos, (const void *)slot})
        if (!aligned(p, 4)) return set_err(FL_B200_ERR_ARG, "paged_plan: misaligned pointer");
    OnDevice on(c->device);
    if (on.err != cudaSuccess) return cuda_err(on.err, "paged_plan: device");
    const PlanArgs a{held, past, fresh, table, free_list, free_in, free_out, q_start, kv_len, pos, slot,
                     c->status + 2, c->status, n_seq, (uint32_t)shift, max_blocks, n_pages, max_tokens};
    const uint32_t grid = std::max(1u, std::min((uint32_t)c->sms, (max_tokens + kPlanThreads - 1) / kPlanThreads));
    return cuda_err(launch_kernel(paged_plan_kernel, dim3(grid), dim3(kPlanThreads), (size_t)3 * (n_seq + 1) * 4, c->stream, true, a), "paged_plan launch");
}

int fl_b200_paged_append(fl_b200_ctx *c, const fl_b200_paged_cache *cache, int act, const void *q, uint32_t n_q, uint32_t q_stride,
                         const void *k, const void *v, uint32_t kv_stride, const int32_t *pos, const int32_t *slot, uint32_t n_tokens,
                         uint32_t n_rot, float freq_base, void *q_out, uint32_t q_out_stride) {
    if (!c) return set_err(FL_B200_ERR_ARG, "paged_append: null context");
    if (int rc = check_cache("paged_append", cache, act)) return rc;
    const uint32_t dim = cache->head_dim;
    if (n_q) {
        if (n_q > 16384) return set_err(FL_B200_ERR_ARG, "paged_append: %u query heads", n_q);
        if (int rc = check_rows("paged_append", "q", q, n_q, dim, q_stride, act)) return rc;
        if (int rc = check_rows("paged_append", "q_out", q_out, n_q, dim, q_out_stride, act)) return rc;
        if (q_out == q && q_out_stride != q_stride) return set_err(FL_B200_ERR_ARG, "paged_append: q in place with two strides");
    }
    if (int rc = check_rows("paged_append", "k", k, cache->n_kv_head, dim, kv_stride, act)) return rc;
    if (int rc = check_rows("paged_append", "v", v, cache->n_kv_head, dim, kv_stride, act)) return rc;
    if (!pos || !slot || !aligned(pos, 4) || !aligned(slot, 4)) return set_err(FL_B200_ERR_ARG, "paged_append: pos or slot is null or misaligned");
    if (n_tokens == 0 || n_tokens >= (1u << 31)) return set_err(FL_B200_ERR_ARG, "paged_append: %u tokens", n_tokens);
    if (n_rot > dim || n_rot % 2) return set_err(FL_B200_ERR_ARG, "paged_append: %u of %u dimensions rotated (an even number)", n_rot, dim);
    if (n_rot && !(std::isfinite(freq_base) && freq_base > 0.f)) return set_err(FL_B200_ERR_ARG, "paged_append: frequency base %g", (double)freq_base);
    OnDevice on(c->device);
    if (on.err != cudaSuccess) return cuda_err(on.err, "paged_append: device");
    AppendArgs a{};
    a.q = q; a.k = k; a.v = v; a.q_out = q_out;
    a.kc = (__half *)cache->k_dev; a.vc = (__half *)cache->v_dev;
    a.pos = pos; a.slot = slot; a.status = c->status;
    a.q_stride = q_stride; a.kv_stride = kv_stride; a.q_out_stride = q_out_stride;
    a.n_q = n_q; a.n_kv = cache->n_kv_head; a.dim_shift = dim == 128 ? 7 : 6; a.n_rot = n_rot;
    a.page_shift = (uint32_t)page_shift_of(cache->page_size); a.n_pages = cache->n_pages;
    // (a product more per pair: 64 roundings of 2^-53 at most)
    const double ratio = n_rot ? std::pow((double)freq_base, -2.0 / n_rot) : 0.0;
    double turn = 1.0 / 6.283185307179586476925;
    for (uint32_t i = 0; i < n_rot / 2; ++i, turn *= ratio) a.turns[i] = turn;
    const uint32_t n_vec = (n_q + 2 * a.n_kv) * dim / (act == FL_B200_ACT_F16 ? 8 : 4);
    const uint32_t y = std::max(1u, std::min((n_vec + kAppThreads - 1) / kAppThreads, 2u * (uint32_t)c->sms / n_tokens));
    const auto kernel = act == FL_B200_ACT_F16 ? paged_append_kernel<__half> : paged_append_kernel<float>;
    const cudaError_t e = launch_kernel(kernel, dim3(n_tokens, y), dim3(kAppThreads), 0, c->stream, true, a);
    return cuda_err(e, "paged_append launch");
}

int fl_b200_paged_attn(fl_b200_ctx *c, const fl_b200_paged_cache *cache, int act, const void *q, uint32_t n_q, uint32_t q_stride,
                       const int32_t *table, uint32_t max_blocks, const int32_t *q_start, const int32_t *kv_len, uint32_t n_seq,
                       uint32_t n_tokens, uint32_t max_new, float scale, void *out, uint32_t out_stride, float *lse_out) {
    if (!c) return set_err(FL_B200_ERR_ARG, "paged_attn: null context");
    if (int rc = check_cache("paged_attn", cache, act)) return rc;
    const uint32_t n_kv = cache->n_kv_head, dim = cache->head_dim, shift = (uint32_t)page_shift_of(cache->page_size);
    if (n_q == 0 || n_q % n_kv || n_q / n_kv > 128)
        return set_err(FL_B200_ERR_ARG, "paged_attn: %u query heads over %u KV heads (whole groups of at most 128)", n_q, n_kv);
    if (int rc = check_rows("paged_attn", "q", q, n_q, dim, q_stride, act)) return rc;
    if (int rc = check_rows("paged_attn", "out", out, n_q, dim, out_stride, act)) return rc;
    if (!table || !q_start || !kv_len || !aligned(table, 4) || !aligned(q_start, 4) || !aligned(kv_len, 4))
        return set_err(FL_B200_ERR_ARG, "paged_attn: table, q_start or kv_len is null or misaligned");
    if (!aligned(lse_out, 8)) return set_err(FL_B200_ERR_ARG, "paged_attn: lse_out must be 8-byte aligned");
    if (n_seq == 0 || n_seq > kPagedMaxSeq) return set_err(FL_B200_ERR_ARG, "paged_attn: %u sequences (1 to %u)", n_seq, kPagedMaxSeq);
    // (a tile of the last key ends within 31 bits)
    if (max_blocks == 0 || ((uint64_t)max_blocks << shift) > (1ull << 31) - 256) return set_err(FL_B200_ERR_ARG, "paged_attn: %u blocks a sequence", max_blocks);
    if (n_tokens == 0 || (uint64_t)n_tokens * (n_q / n_kv) >= (1ull << 31)) return set_err(FL_B200_ERR_ARG, "paged_attn: %u tokens", n_tokens);
    if (max_new == 0 || max_new > n_tokens) return set_err(FL_B200_ERR_ARG, "paged_attn: max_new %u of %u tokens", max_new, n_tokens);
    if (!(std::isfinite(scale) && scale > 0.f)) return set_err(FL_B200_ERR_ARG, "paged_attn: scale %g (positive)", (double)scale);
    OnDevice on(c->device);
    if (on.err != cudaSuccess) return cuda_err(on.err, "paged_attn: device");
    if (!c->paged_part) {
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        if (const cudaError_t e = cudaStreamIsCapturing(c->stream, &cap)) return cuda_err(e, "paged_attn: capture status");
        if (cap != cudaStreamCaptureStatusNone)
            return set_err(FL_B200_ERR_STATE, "paged_attn: the first call on a context allocates its scratch; make it before a capture");
        void *part = nullptr, *tickets = nullptr;
        cudaError_t e = cudaMalloc(&part, paged_few_part_bytes(c->sms) + paged_tm_part_bytes(c->sms));
        if (e == cudaSuccess) e = cudaMalloc(&tickets, kPagedTickets * sizeof(uint32_t));
        if (e == cudaSuccess) e = cudaMemsetAsync(tickets, 0, kPagedTickets * sizeof(uint32_t), c->stream);
        if (e != cudaSuccess) {
            cudaFree(part);
            cudaFree(tickets);
            cudaGetLastError();
            return cuda_err(e, "paged_attn: scratch");
        }
        c->paged_part = (float *)part;
        c->paged_tickets = (uint32_t *)tickets;
    }
    PagedAttnArgs a{};
    a.q = q; a.out = out; a.lse = reinterpret_cast<float2 *>(lse_out);
    a.table = table; a.q_start = q_start; a.kv_len = kv_len;
    a.part = c->paged_part; a.tickets = c->paged_tickets; a.status = c->status;
    a.q_stride = q_stride; a.out_stride = out_stride;
    a.n_seq = n_seq; a.max_blocks = max_blocks; a.n_tokens = n_tokens; a.max_new = max_new;
    a.n_pages = cache->n_pages; a.page_shift = shift;
    a.n_kv = n_kv; a.group = n_q / n_kv; a.half = act == FL_B200_ACT_F16 ? 1u : 0u;
    a.scale = scale;
    a.part_tm = c->paged_part + paged_few_part_bytes(c->sms) / sizeof(float);
    const bool many = (uint64_t)max_new * a.group > kFewRows;
    a.spare = !many ? 0 : a.half && dim == 128 ? kSpareHalf128 : kSpare;
    if (many && n_seq <= 32 && (uint64_t)n_seq * n_kv * (((uint64_t)max_blocks << shift) / 128 + kSpareStart) <= kSpareNoLaunch) a.spare = kSpareAll;
    if (a.spare != kSpareAll)
        if (int rc = cuda_err(launch_paged_few(a, cache->k_dev, cache->v_dev, dim, c->sms, c->stream), "paged_attn launch")) return rc;
    return many ? cuda_err(launch_paged_tm(a, cache->k_dev, cache->v_dev, dim, c->sms, c->stream), "paged_attn launch") : FL_B200_OK;
}

} // extern "C"
