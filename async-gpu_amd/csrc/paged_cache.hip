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
    PageDiv div;
};

constexpr int PLAN_THREADS = 256, PLAN_WAVES = PLAN_THREADS / 64;

struct PlanSums {
    long long freed, pages, tokens;
    __device__ __forceinline__ void add(const PlanSums &o) {
        freed += o.freed;
        pages += o.pages;
        tokens += o.tokens;
    }
};
__device__ __forceinline__ long long shift_up(long long v, int by, int lane) {
    const long long o = __shfl_up(v, by, kWave);
    return lane >= by ? o : 0;
}

// What a request asks for: its positions so far, the pages that they are on, new tokens and pages (none where its table row is too short).
struct Ask {
    int cached, have, tokens, pages;
    bool ended;
    __device__ __forceinline__ Ask(const PlanArgs &p, int b) {
        const int n = p.new_lens[b];
        cached = min(max(p.cached_lens[b], 0), p.width * p.div.size);
        ended = n < 0;
        have = (int)(((long long)cached + p.div.size - 1) / p.div.size);
        const long long total = (long long)cached + max(n, 0);
        const bool fits = !ended && total <= (long long)p.width * p.div.size;
        tokens = fits ? n : 0;
        pages = fits ? (int)((total + p.div.size - 1) / p.div.size) - have : 0;
    }
};

// The last entry of at[0 .. n - 1] (ascending, at[0] = 0) that is not above x.
__device__ __forceinline__ int entry_of(const int *at, int n, int x) {
    int lo = 0;
    for (int step = 1 << (31 - __builtin_clz(n)); step > 0; step >>= 1) lo = lo + step < n && at[lo + step] <= x ? lo + step : lo;
    return lo;
}

// Every workgroup adds up all requests for itself (they are few, and nobody waits for anybody), then the workgroups share what there is to write.
// Nothing is read that another one writes: table entries of pages held so far, and the stack below n_free; new pages are looked up where they
// came from.  What bounds it: a chain of loads, sums and searches, 16 bytes a token at the largest.
__global__ __launch_bounds__(PLAN_THREADS) void paged_plan_kernel(const PlanArgs p) {
    extern __shared__ int s_plan[];  // of every request: pages freed before it, pages taken before it, tokens before it
    __shared__ PlanSums s_wave[PLAN_WAVES];
    __shared__ long long s_used[2][PLAN_WAVES];
    int *const s_freed = s_plan, *const s_pages = s_plan + p.batch, *const s_start = s_plan + 2 * p.batch;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int each = (p.batch + PLAN_THREADS - 1) / PLAN_THREADS, b0 = tid * each, b1 = min(b0 + each, p.batch);
    const int n_free = min(max(*p.n_free, 0), p.stack_size);
    PlanSums mine = {0, 0, 0};
    for (int b = b0; b < b1; ++b) {
        const Ask a(p, b);
        mine.add({a.ended ? a.have : 0, a.pages, a.tokens});
    }
    PlanSums run = mine;
#pragma unroll
    for (int by = 1; by < 64; by <<= 1) run.add({shift_up(run.freed, by, lane), shift_up(run.pages, by, lane), shift_up(run.tokens, by, lane)});
    if (lane == 63) s_wave[wave] = run;
    __syncthreads();
    run.add({-mine.freed, -mine.pages, -mine.tokens});
    PlanSums all = {0, 0, 0};
#pragma unroll
    for (int w = 0; w < PLAN_WAVES; ++w) {
        if (w < wave) run.add(s_wave[w]);
        all.add(s_wave[w]);
    }
    const int top = (int)min((long long)n_free + all.freed, (long long)p.stack_size);  // the stack with what was freed on it
    // Requests are served while the sums with their own are within what there is; sums only grow, so that the first one that is not is the last.
    long long used_pages = 0, used_tokens = 0;
    {
        PlanSums at = run;
        for (int b = b0; b < b1; ++b) {
            const Ask a(p, b);
            at.add({a.ended ? a.have : 0, a.pages, a.tokens});
            if (at.pages <= top && at.tokens <= p.max_tokens) used_pages = at.pages, used_tokens = at.tokens;
        }
    }
#pragma unroll
    for (int by = 32; by > 0; by >>= 1) {
        used_pages = max(used_pages, __shfl_xor(used_pages, by, kWave));
        used_tokens = max(used_tokens, __shfl_xor(used_tokens, by, kWave));
    }
    if (lane == 0) s_used[0][wave] = used_pages, s_used[1][wave] = used_tokens;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PLAN_WAVES; ++w) {
        used_pages = max(used_pages, s_used[0][w]);
        used_tokens = max(used_tokens, s_used[1][w]);
    }
    const int taken = (int)used_pages, tokens = (int)used_tokens, left = top - taken;
    const bool writes = blockIdx.x == 0;
    for (int b = b0; b < b1; ++b) {
        const Ask a(p, b);
        const PlanSums before = run;
        run.add({a.ended ? a.have : 0, a.pages, a.tokens});
        const bool served = run.pages <= top && run.tokens <= p.max_tokens;
        s_freed[b] = (int)min(before.freed, (long long)INT32_MAX);
        s_pages[b] = (int)min(before.pages, used_pages);
        s_start[b] = (int)min(before.tokens, used_tokens);
        if (writes) {
            p.kv_lens[b] = a.ended ? 0 : a.cached + (served ? a.tokens : 0);
            p.query_start[b] = s_start[b];
        }
    }
    if (writes && tid == 0) {
        p.query_start[p.batch] = tokens;
        *p.n_free_out = left;
    }
    __syncthreads();
    const int at = blockIdx.x * PLAN_THREADS + tid, stride = gridDim.x * PLAN_THREADS;
    auto freed_page = [&](int i) {
        const int b = entry_of(s_freed, p.batch, i);
        return p.tables[(size_t)b * p.width + (i - s_freed[b])];
    };
    auto new_page = [&](int i) {  // page i that this step takes
        const int place = top - 1 - i;
        return place < n_free ? p.free_pages[place] : freed_page(place - n_free);
    };
    for (int i = at; i < max(taken, left - n_free); i += stride) {
        if (i < taken) {
            const int b = entry_of(s_pages, p.batch, i), have = p.div.page(min(max(p.cached_lens[b], 0), p.width * p.div.size) + p.div.size - 1);
            p.tables[(size_t)b * p.width + have + (i - s_pages[b])] = new_page(i);
        }
        if (i < left - n_free) p.free_pages[n_free + i] = freed_page(i);
    }
    for (int t = at; t < p.max_tokens; t += stride) {
        int slot = -1, pos = 0;
        if (t < tokens) {
            const int b = entry_of(s_start, p.batch, t), cached = min(max(p.cached_lens[b], 0), p.width * p.div.size);
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

// 16 bytes of K and of V a thread, 16 or 8 threads a row of 64.
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
    const PlanArgs p = {cached_lens, new_lens, n_free, block_tables, free_pages, kv_lens, query_start, slots, positions, n_free_out, batch, table_width, stack_size,
                        max_tokens, PageDiv::of(page_size)};
    const int wgs = std::max(1, std::min(ceil_div(std::max(max_tokens, batch), 4 * PLAN_THREADS), ctx->num_cus));
    hipLaunchKernelGGL(paged_plan_kernel, dim3(wgs), dim3(PLAN_THREADS), (3 * batch + 1) * sizeof(int), ctx->stream, p);
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
