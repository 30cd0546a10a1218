// Bookkeeping of a KV cache in pages on the device, and the K and V rows of new tokens on their way into it.
#include "agpu_internal.h"
#include "paged.h"

#include <algorithm>

namespace {

using paged::PageDiv;

struct PlanArgs {
    const int *cached_lens, *new_lens, *n_free;
    int *tables, *free_pages;
    int *kv_lens, *query_start, *slots, *positions, *n_free_out;
    int batch, width, stack_size, max_tokens;
    int page_groups;  // workgroups that write pages; the others write slots and positions (one alone: both)
    PageDiv div;
};

constexpr int PLAN_THREADS = 256, PLAN_WAVES = PLAN_THREADS / 64;

// Sums that stay at their largest value once they reach it (what they are compared with is below 2^31).
struct PlanSums {
    uint32_t freed, pages, tokens;
    __device__ __forceinline__ void add(const PlanSums &o) {
        freed = __builtin_elementwise_add_sat(freed, o.freed);
        pages = __builtin_elementwise_add_sat(pages, o.pages);
        tokens = __builtin_elementwise_add_sat(tokens, o.tokens);
    }
    template <int CTRL, int ROWS>
    __device__ __forceinline__ void add_moved() {
        auto move = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); };
        add({move(freed), move(pages), move(tokens)});
    }
    // over the lanes up to this one
    __device__ __forceinline__ void scan() {
        add_moved<0x111, 0xf>();  // row_shr 1, 2, 4, 8: within rows of 16
        add_moved<0x112, 0xf>();
        add_moved<0x114, 0xf>();
        add_moved<0x118, 0xf>();
        add_moved<0x142, 0xa>();  // row_bcast 15: row 0 to 1, 2 to 3
        add_moved<0x143, 0xc>();  // row_bcast 31: rows 0 and 1 to 2 and 3
    }
};

// What a request asks for: its positions so far, the pages that they are on, new tokens and pages (none where its table row is too short).
struct Ask {
    int cached, have, tokens, pages;
    bool ended;
    __device__ __forceinline__ Ask() : cached(0), have(0), tokens(0), pages(0), ended(false) {}
    __device__ __forceinline__ Ask(const PlanArgs &p, int cached_, int n) {
        const int held = p.width * p.div.size;
        cached = min(max(cached_, 0), held);
        ended = n < 0;
        have = p.div.page(cached + p.div.size - 1);
        const bool fits = !ended && n <= held - cached;
        tokens = fits ? n : 0;
        pages = fits ? p.div.page(cached + n + p.div.size - 1) - have : 0;
    }
    __device__ __forceinline__ PlanSums sums() const { return {ended ? (uint32_t)have : 0u, (uint32_t)pages, (uint32_t)tokens}; }
};

// The last entry of at[0 .. n - 1] (ascending, at[0] = 0) that is not above x.
__device__ __forceinline__ int entry_of(const int *at, int n, int x) {
    int lo = 0;
    for (int step = 1 << (31 - __builtin_clz(n)); step > 0; step >>= 1) lo = lo + step < n && at[lo + step] <= x ? lo + step : lo;
    return lo;
}

// Every workgroup adds up all requests for itself (they are few, and nobody waits for anybody), then the workgroups share what there is to write.
// Nothing is read that another one writes: table entries of pages held so far, and the stack below n_free; new pages are looked up where they
// came from.  What bounds it: a chain of loads, sums and searches, 16 bytes a token at the largest.  8 requests 2.8 us (4.9 a call from Python, which is what
// the host takes), 512 requests with up to 200 new tokens each 5.8 (7.7 where every workgroup has pages and tokens).
// EACH: requests of a thread.
template <int EACH>
__global__ __launch_bounds__(PLAN_THREADS) void paged_plan_kernel(const PlanArgs p) {
    constexpr bool kept = EACH <= 4;  // positions so far in LDS too (16 requests a thread would be too many)
    extern __shared__ int s_plan[];   // of every request: pages freed before it, pages taken before it, tokens before it, positions so far
    __shared__ PlanSums s_wave[PLAN_WAVES];
    __shared__ uint32_t s_used[2][PLAN_WAVES];
    int *const s_freed = s_plan, *const s_pages = s_plan + p.batch, *const s_start = s_plan + 2 * p.batch, *const s_cached = s_plan + 3 * p.batch;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b0 = tid * EACH;
    int cached[EACH], fresh[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        cached[e] = b0 + e < p.batch ? p.cached_lens[b0 + e] : 0;
        fresh[e] = b0 + e < p.batch ? p.new_lens[b0 + e] : 0;
    }
    const int n_free = min(max(*p.n_free, 0), p.stack_size);
    Ask ask[EACH];
    PlanSums run = {0, 0, 0};
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        ask[e] = Ask(p, cached[e], fresh[e]);
        run.add(ask[e].sums());
    }
    run.scan();
    if (lane == 63) s_wave[wave] = run;
    // the lanes before this one
    PlanSums before = {(uint32_t)__shfl_up((int)run.freed, 1, kWave), (uint32_t)__shfl_up((int)run.pages, 1, kWave), (uint32_t)__shfl_up((int)run.tokens, 1, kWave)};
    if (lane == 0) before = {0, 0, 0};
    __syncthreads();
    uint32_t freed = 0;
#pragma unroll
    for (int w = 0; w < PLAN_WAVES; ++w) {
        if (w < wave) before.add(s_wave[w]);
        freed = __builtin_elementwise_add_sat(freed, s_wave[w].freed);
    }
    const uint32_t top = min(__builtin_elementwise_add_sat((uint32_t)n_free, freed), (uint32_t)p.stack_size);  // the stack with what was freed on it
    // Requests are served while the sums with their own are within what there is; sums only grow, so that the first one that is not is the last.
    uint32_t used_pages = 0, used_tokens = 0;
    run = before;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        run.add(ask[e].sums());
        if (run.pages <= top && run.tokens <= (uint32_t)p.max_tokens) used_pages = run.pages, used_tokens = run.tokens;
    }
    used_pages = wave_minmax_u32<true>(used_pages);
    used_tokens = wave_minmax_u32<true>(used_tokens);
    if (lane == 0) s_used[0][wave] = used_pages, s_used[1][wave] = used_tokens;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PLAN_WAVES; ++w) {
        used_pages = max(used_pages, s_used[0][w]);
        used_tokens = max(used_tokens, s_used[1][w]);
    }
    const int taken = (int)used_pages, tokens = (int)used_tokens, left = (int)top - taken;
    const bool writes = blockIdx.x == 0;
    run = before;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int b = b0 + e;
        if (b >= p.batch) break;
        if (kept) s_cached[b] = ask[e].cached;
        s_freed[b] = (int)min(run.freed, (uint32_t)INT32_MAX);
        s_pages[b] = (int)min(run.pages, used_pages);
        s_start[b] = (int)min(run.tokens, used_tokens);
        run.add(ask[e].sums());
        if (writes) {
            const bool served = run.pages <= top && run.tokens <= (uint32_t)p.max_tokens;
            p.kv_lens[b] = ask[e].ended ? 0 : ask[e].cached + (served ? ask[e].tokens : 0);
            p.query_start[b] = s_start[b];
        }
    }
    if (writes && tid == 0) {
        p.query_start[p.batch] = tokens;
        *p.n_free_out = left;
    }
    __syncthreads();
    // pages and tokens by workgroups of their own, each a chain of searches and loads, unless a single one does it all
    const bool for_pages = (int)blockIdx.x < p.page_groups, for_tokens = !for_pages || gridDim.x == 1;
    const int at = ((int)blockIdx.x - (for_pages ? 0 : p.page_groups)) * PLAN_THREADS + tid;
    const int stride = (for_pages ? p.page_groups : (int)gridDim.x - p.page_groups) * PLAN_THREADS;
    auto positions = [&](int b) { return kept ? s_cached[b] : min(max(p.cached_lens[b], 0), p.width * p.div.size); };
    auto freed_page = [&](int i) {
        const int b = entry_of(s_freed, p.batch, i);
        return p.tables[(size_t)b * p.width + (i - s_freed[b])];
    };
    auto new_page = [&](int i) {  // page i that this step takes
        const int place = (int)top - 1 - i;
        return place < n_free ? p.free_pages[place] : freed_page(place - n_free);
    };
    for (int i = at; for_pages && i < max(taken, left - n_free); i += stride) {
        if (i < taken) {
            const int b = entry_of(s_pages, p.batch, i), have = p.div.page(positions(b) + p.div.size - 1);
            p.tables[(size_t)b * p.width + have + (i - s_pages[b])] = new_page(i);
        }
        if (i < left - n_free) p.free_pages[n_free + i] = freed_page(i);
    }
    for (int t = at; for_tokens && t < p.max_tokens; t += stride) {
        int slot = -1, pos = 0;
        if (t < tokens) {
            const int b = entry_of(s_start, p.batch, t), cached = positions(b);
            pos = cached + (t - s_start[b]);
            const int k = p.div.page(pos), have = p.div.page(cached + p.div.size - 1);
            const int page = k < have ? p.tables[(size_t)b * p.width + k] : new_page(s_pages[b] + k - have);
            const long long to = (long long)page * p.div.size + (pos - k * p.div.size);
            slot = page >= 0 && to <= INT32_MAX ? (int)to : -1;
        }
        p.slots[t] = slot;
        p.positions[t] = pos;
    }
}

struct AppendArgs {
    const float *k, *v;
    long long k_token, k_head, v_token, v_head;
    char *k_cache, *v_cache;
    long long k_page, v_page;
    const int *slots;
    int rows, slots_all;  // rows: tokens * heads
    PageDiv heads, div;
};

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {  // to nearest, ties to even; NaN stays NaN
    auto one = [](float x) { return x != x ? 0x7fc0u : (__float_as_uint(x) + 0x7fffu + ((__float_as_uint(x) >> 16) & 1u)) >> 16; };
    return one(a) | one(b) << 16;
}
__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
    return (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)a) | (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)b) << 16;
}
template <int TYPE>
__device__ __forceinline__ uint4 packed(const float *from) {  // 16 bytes of the cache
    const float4 a = load4(from);
    if (TYPE == AGPU_CACHE_F32) return __builtin_bit_cast(uint4, a);
    const float4 b = load4(from + 4);
    if (TYPE == AGPU_CACHE_BF16) return make_uint4(bf16_pair(a.x, a.y), bf16_pair(a.z, a.w), bf16_pair(b.x, b.y), bf16_pair(b.z, b.w));
    return make_uint4(f16_pair(a.x, a.y), f16_pair(a.z, a.w), f16_pair(b.x, b.y), f16_pair(b.z, b.w));
}

// 16 bytes of K and of V a thread, 16 or 8 threads a row of 64.  Bound by the bytes: 4096 rows of 25 heads to bf16 (79 MB) 13.7 us, 5.7 TB/s; 16 rows of 12 heads 2.4 us
// (3.9 a call from Python).
template <int TYPE>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs p) {
    constexpr int EL = TYPE == AGPU_CACHE_F32 ? 4 : 8, LANES = 64 / EL;
    const int row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, sub = threadIdx.x % LANES;
    if (row >= p.rows) return;
    const int t = p.heads.page(row), h = row - t * p.heads.size, slot = p.slots[t];
    if ((unsigned)slot >= (unsigned)p.slots_all) return;
    const uint4 k = packed<TYPE>(p.k + (long long)t * p.k_token + (long long)h * p.k_head + EL * sub);
    const uint4 v = packed<TYPE>(p.v + (long long)t * p.v_token + (long long)h * p.v_head + EL * sub);
    const int page = p.div.page(slot);
    const long long at = (long long)(h * p.div.size + (slot - page * p.div.size)) * 64 + EL * sub;
    *reinterpret_cast<uint4 *>(p.k_cache + (page * p.k_page + at) * (16 / EL)) = k;
    *reinterpret_cast<uint4 *>(p.v_cache + (page * p.v_page + at) * (16 / EL)) = v;
}

}  // namespace

AGPU_EXPORT int32_t agpu_paged_plan(agpu_ctx *ctx, const int32_t *cached_lens, const int32_t *new_lens, int32_t *block_tables, int32_t *free_pages,
                                    const int32_t *n_free, int32_t *kv_lens, int32_t *query_start, int32_t *slots, int32_t *positions,
                                    int32_t *n_free_out, int32_t batch, int32_t table_width, int32_t stack_size, int32_t page_size,
                                    int32_t max_tokens) {
    AGPU_REQUIRE_CTX(ctx);
    const paged::Refusal no = paged::refuse_plan(batch, table_width, stack_size, page_size, max_tokens);
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_plan: %s", no.why);
    if ((batch > 0 && (!cached_lens || !new_lens || !kv_lens || (!block_tables && table_width > 0))) || (!free_pages && stack_size > 0) || !n_free || !query_start ||
        !n_free_out || (max_tokens > 0 && (!slots || !positions)))
        return agpu_fail(ctx, AGPU_ERR_NULL_POINTER, "paged_plan: null pointer");
    if ((batch > 0 && (kv_lens == cached_lens || kv_lens == new_lens)) || n_free_out == n_free)
        return agpu_fail(ctx, AGPU_ERR_UNSUPPORTED, "paged_plan: the outputs do not overlap the inputs");
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    // as many workgroups as find a CU each; of the pages as many as the tokens could fill
    auto groups = [](int64_t work, int most) { return (int)std::max<int64_t>(1, std::min<int64_t>((work + PLAN_THREADS - 1) / PLAN_THREADS, most)); };
    const int page_groups = groups((int64_t)max_tokens / page_size + batch, ctx->num_cus / 4), token_groups = max_tokens <= PLAN_THREADS && page_groups == 1 ? 0 : groups(max_tokens, ctx->num_cus - page_groups);
    const PlanArgs p = {cached_lens, new_lens, n_free, block_tables, free_pages, kv_lens, query_start, slots, positions, n_free_out, batch, table_width, stack_size,
                        max_tokens, page_groups, PageDiv::of(page_size)};
    const size_t lds = ((batch <= 4 * PLAN_THREADS ? 4 : 3) * batch + 1) * sizeof(int);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(page_groups + token_groups), dim3(PLAN_THREADS), lds, ctx->stream, p); };
    static_assert(paged::kMaxRequests <= 16 * PLAN_THREADS && 3 * paged::kMaxRequests * sizeof(int) <= 65536 - 1024, "");
    if (batch <= PLAN_THREADS) go(paged_plan_kernel<1>);
    else if (batch <= 4 * PLAN_THREADS) go(paged_plan_kernel<4>);
    else go(paged_plan_kernel<16>);
    return AGPU_LAUNCH_CHECK(ctx, "paged_plan_kernel");
}

AGPU_EXPORT int32_t agpu_paged_kv_append(agpu_ctx *ctx, const float *k, const float *v, int64_t k_token_stride, int64_t k_head_stride,
                                         int64_t v_token_stride, int64_t v_head_stride, void *k_cache, void *v_cache, int64_t k_page_stride,
                                         int64_t v_page_stride, const int32_t *slots, int32_t tokens, int32_t n_kv_heads, int32_t n_pages,
                                         int32_t page_size, int32_t d_head, int32_t cache_type) {
    AGPU_REQUIRE_CTX(ctx);
    paged::Refusal no = paged::refuse_cache((uintptr_t)k_cache, (uintptr_t)v_cache, k_page_stride, v_page_stride, n_kv_heads, n_pages, page_size, d_head, cache_type);
    if (no.code == AGPU_OK) no = paged::refuse_append(tokens, n_kv_heads);
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_kv_append: %s", no.why);
    if (tokens == 0) return AGPU_OK;
    if (!k || !v || !k_cache || !v_cache || !slots) return agpu_fail(ctx, AGPU_ERR_NULL_POINTER, "paged_kv_append: null pointer");
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    const AppendArgs p = {k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, static_cast<char *>(k_cache), static_cast<char *>(v_cache), k_page_stride,
                          v_page_stride, slots, tokens * n_kv_heads, n_pages * page_size, PageDiv::of(n_kv_heads), PageDiv::of(page_size)};
    auto go = [&](auto kernel, int lanes) { hipLaunchKernelGGL(kernel, dim3(ceil_div(p.rows, 256 / lanes)), dim3(256), 0, ctx->stream, p); };
    if (cache_type == AGPU_CACHE_F32) go(paged_append_kernel<AGPU_CACHE_F32>, 16);
    else if (cache_type == AGPU_CACHE_F16) go(paged_append_kernel<AGPU_CACHE_F16>, 8);
    else go(paged_append_kernel<AGPU_CACHE_BF16>, 8);
    return AGPU_LAUNCH_CHECK(ctx, "paged_append_kernel");
}
