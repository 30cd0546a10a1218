// A KV cache cut down to a budget: which places of a request keep their keys, and the pages behind them.
//
// paged_evict_kernel, a workgroup a request and K/V head: weights as integers in the order of the floats, the smallest one that stays found bit by bit from the top (two a step, by
// counting), equal ones in the order of their places.  Those that stay keep their places, except where that is behind what is kept: these move into places of evicted ones, the first to the
// first.  So no more is moved than has to be, sources and targets never overlap, and nothing waits for the order of moves.
#include "agpu_internal.h"
#include "paged.h"

#include <algorithm>

namespace {

using paged::PageDiv;

struct EvictArgs {
    char *k, *v;
    long long k_page, v_page;  // bytes between pages
    float *weights;
    long long w_page;  // elements
    const int *tables, *kv_lens;
    int n_kv, n_pages, width, held, limit, keep, recent, sinks;
    PageDiv div;
};

// Positions of a thread that are in registers at a time: position e * 512 + tid of a block.
constexpr int kEvictThreads = 512, kEvictWaves = kEvictThreads / 64, kEvictEach = 8, kEvictListed = 1024;

// Larger for larger weights; zeros of both signs are equal; no number is less than all numbers, and a page outside the cache (0) less than that.
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    return w != w ? 1u : (u >> 31) ? ~u : u | 0x80000000u;
}

struct EvictShared {
    int counts[2][kEvictWaves][3];
    int ties[kEvictEach * kEvictWaves];  // of each 64 positions of a block: how many weigh the least
    int before[kEvictThreads], wave_sums[kEvictWaves];
    int to[kEvictListed], from[kEvictListed];  // positions
};

// Set bits of `which` below this lane.
__device__ __forceinline__ int bits_below(uint64_t which) { return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(which >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)which, 0)); }
__device__ __forceinline__ uint64_t first_bits(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }

// ROW: 16-byte pieces of a row of K or V.  stays: a bit for each position of a request.
template <int ROW>
__global__ __launch_bounds__(kEvictThreads) void paged_evict_kernel(const EvictArgs p) {
    extern __shared__ uint64_t stays[];
    __shared__ EvictShared s;
    const int b = blockIdx.x / p.n_kv, h = blockIdx.x - b * p.n_kv, n = max(min(p.kv_lens[b], p.held), 0);
    if (n <= p.limit) return;
    constexpr int BLOCK = kEvictThreads * kEvictEach;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int *table = p.tables + (size_t)b * p.width;
    const int blocks = (n + BLOCK - 1) / BLOCK, chunks = (n + 63) / 64, need = p.keep - p.sinks - p.recent;
    auto slot_of = [&](int i, int &page) {  // where position i is on its page; -1: the page is outside the cache
        const int at = p.div.page(i);
        page = table[at];
        return (unsigned)page < (unsigned)p.n_pages ? h * p.div.size + (i - at * p.div.size) : -1;
    };
    auto middle = [&](int i) { return i >= p.sinks && i < n - p.recent; };
    uint32_t key[kEvictEach];
    auto load = [&](int block) {
        int page[kEvictEach], slot[kEvictEach];
#pragma unroll
        for (int e = 0; e < kEvictEach; ++e) {
            const int i = block * BLOCK + e * kEvictThreads + tid;
            slot[e] = -1;
            if (middle(i)) slot[e] = slot_of(i, page[e]);
        }
#pragma unroll
        for (int e = 0; e < kEvictEach; ++e) key[e] = slot[e] >= 0 ? order_of(p.weights[page[e] * p.w_page + slot[e]]) : 0;
    };
    load(0);
    // The largest `least` that has `need` keys or more from it on.
    uint32_t least = need > 0 ? 0u : 0xffffffffu;
    bool exact = need == 0;  // just as many
    for (int bit = 30; bit >= 0 && !exact; bit -= 2) {
        int count[3] = {0, 0, 0};
        for (int block = 0; block < blocks; ++block) {
            if (blocks > 1) load(block);
#pragma unroll
            for (int e = 0; e < kEvictEach; ++e)
#pragma unroll
                for (int c = 0; c < 3; ++c) count[c] += __popcll(__ballot(key[e] >= (least | (uint32_t)(c + 1) << bit)));
        }
        int(&counts)[kEvictWaves][3] = s.counts[bit >> 1 & 1];  // (what the other one holds has been read before the next barrier)
        if (lane == 0)
#pragma unroll
            for (int c = 0; c < 3; ++c) counts[wave][c] = count[c];
        __syncthreads();
        int all[3] = {0, 0, 0};
#pragma unroll
        for (int w = 0; w < kEvictWaves; ++w)
#pragma unroll
            for (int c = 0; c < 3; ++c) all[c] += counts[w][c];
        const uint32_t low = least;
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (all[c] >= need) {
                least = low | (uint32_t)(c + 1) << bit;
                exact = all[c] == need;
            }
    }
    int ties = 0;  // how many of those that weigh the least stay: the first ones
    if (!exact) {
        int more = 0;
        for (int block = 0; block < blocks; ++block) {
            if (blocks > 1) load(block);
#pragma unroll
            for (int e = 0; e < kEvictEach; ++e) more += __popcll(__ballot(key[e] > least));
        }
        __syncthreads();
        if (lane == 0) s.counts[0][wave][0] = more;
        __syncthreads();
        ties = need;
#pragma unroll
        for (int w = 0; w < kEvictWaves; ++w) ties -= s.counts[0][w][0];
    }
    // Who stays, a bit a position.
    for (int block = 0; block < blocks; ++block) {
        if (blocks > 1) load(block);
        uint64_t equal[kEvictEach];
        int before = 0, all = 0;
        if (!exact) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kEvictEach; ++e) {
                equal[e] = __ballot(middle(block * BLOCK + e * kEvictThreads + tid) && key[e] == least);
                if (lane == 0) s.ties[e * kEvictWaves + wave] = __popcll(equal[e]);
            }
            __syncthreads();
            static_assert(kEvictEach * kEvictWaves == 64, "");
            const int own = s.ties[lane];
            before = wave_running_sum(own);
            all = __builtin_amdgcn_readlane(before, 63);
            before -= own;
        }
#pragma unroll
        for (int e = 0; e < kEvictEach; ++e) {
            const int i = block * BLOCK + e * kEvictThreads + tid;
            bool stay = i < n && (!middle(i) || key[e] > least);
            if (exact) stay = stay || (middle(i) && key[e] == least);
            else if (middle(i) && key[e] == least) stay = __builtin_amdgcn_readlane(before, e * kEvictWaves + __builtin_amdgcn_readfirstlane(wave)) + bits_below(equal[e]) < ties;
            const uint64_t word = __ballot(stay);
            const int chunk = (block * kEvictEach + e) * kEvictWaves + wave;
            if (lane == 0 && chunk < chunks) stays[chunk] = word;
        }
        ties -= all;
    }
    __syncthreads();
    // Of 64 positions those that are evicted and get another one's key, or those that move.
    auto word = [&](bool hole, int chunk) {
        const uint64_t kept = first_bits(p.keep - 64 * chunk), stay = stays[chunk];
        return hole ? ~stay & kept : stay & ~kept;
    };
    int moves = 0;  // as many as places of evicted ones
    for (int chunk = tid; chunk < chunks; chunk += kEvictThreads) moves += __popcll(word(false, chunk));
    moves = __builtin_amdgcn_readlane(wave_running_sum(moves), 63);
    if (lane == 0) s.wave_sums[wave] = moves;
    __syncthreads();
    moves = 0;
#pragma unroll
    for (int w = 0; w < kEvictWaves; ++w) moves += s.wave_sums[w];
    __syncthreads();
    // Numbers done .. done + kEvictListed - 1 of one kind, from the chunks `first` on, before which there are `base`.
    auto list = [&](bool hole, int done, int &first, int &base, int *out) {
        for (;;) {
            const int chunk = first + tid, count = chunk < chunks ? __popcll(word(hole, chunk)) : 0, upto = wave_running_sum(count);
            if (lane == 63) s.wave_sums[wave] = upto;
            __syncthreads();
            int before = base - done + upto - count, all = 0;
#pragma unroll
            for (int w = 0; w < kEvictWaves; ++w) {
                if (w < wave) before += s.wave_sums[w];
                all += s.wave_sums[w];
            }
            s.before[tid] = before;
            __syncthreads();
            for (int c = wave; c < kEvictThreads && first + c < chunks; c += kEvictWaves) {
                const int rank = s.before[c];
                if (rank >= kEvictListed) break;
                const uint64_t bits = word(hole, first + c);
                const int mine = rank + bits_below(bits);
                if ((bits >> lane & 1) && mine >= 0 && mine < kEvictListed) out[mine] = 64 * (first + c) + lane;
            }
            __syncthreads();
            if (base + all >= done + kEvictListed || first + kEvictThreads >= chunks) return;
            first += kEvictThreads;
            base += all;
        }
    };
    int first_hole = 0, holes_before = 0, first_move = 0, moves_before = 0;
    for (int done = 0; done < moves; done += kEvictListed) {
        list(true, done, first_hole, holes_before, s.to);
        list(false, done, first_move, moves_before, s.from);
        const int now = min(moves - done, kEvictListed);
        constexpr int ROUNDS = 4;
        for (int base = 0; base < now * ROW; base += ROUNDS * kEvictThreads) {
            uint4 kx[ROUNDS], vx[ROUNDS];
            float w[ROUNDS];
            int from_page[ROUNDS], to_page[ROUNDS], from[ROUNDS], to[ROUNDS], piece[ROUNDS];
            bool ok[ROUNDS];
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r) {
                const int i = base + r * kEvictThreads + tid, m = min(i / ROW, now - 1);
                piece[r] = i % ROW;
                from[r] = slot_of(s.from[m], from_page[r]);
                to[r] = slot_of(s.to[m], to_page[r]);
                ok[r] = i < now * ROW && from[r] >= 0 && to[r] >= 0;
            }
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r)
                if (ok[r]) {
                    const long long at = ((long long)from[r] * ROW + piece[r]) * 16;
                    kx[r] = *reinterpret_cast<const uint4 *>(p.k + from_page[r] * p.k_page + at);
                    vx[r] = *reinterpret_cast<const uint4 *>(p.v + from_page[r] * p.v_page + at);
                    if (piece[r] == 0) w[r] = p.weights[from_page[r] * p.w_page + from[r]];
                }
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r)
                if (ok[r]) {
                    const long long at = ((long long)to[r] * ROW + piece[r]) * 16;
                    *reinterpret_cast<uint4 *>(p.k + to_page[r] * p.k_page + at) = kx[r];
                    *reinterpret_cast<uint4 *>(p.v + to_page[r] * p.v_page + at) = vx[r];
                    if (piece[r] == 0) p.weights[to_page[r] * p.w_page + to[r]] = w[r];
                }
        }
        __syncthreads();  // the lists
    }
}

// ---- lengths and pages ----------------------------------------------------------------------------

struct TrimArgs {
    const int *kv_lens, *tables, *n_free;
    int *free_pages, *kv_out, *evicted, *n_free_out;
    int batch, width, stack_size, limit, keep;
    PageDiv div;
};

constexpr int TRIM_THREADS = 256;

// Every workgroup adds up the pages of all requests for itself, then they share the stack's new entries.
__global__ __launch_bounds__(TRIM_THREADS) void paged_trim_kernel(const TrimArgs p) {
    extern __shared__ int s_start[];  // pages given back before each request, and all
    __shared__ uint32_t s_wave[TRIM_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int each = (p.batch + TRIM_THREADS - 1) / TRIM_THREADS, b0 = tid * each, held = p.width * p.div.size;
    auto pages = [&](int n) { return p.div.page(n + p.div.size - 1); };
    auto given = [&](int b) {
        const int n = max(min(p.kv_lens[b], held), 0);
        return n > p.limit ? pages(n) - pages(p.keep) : 0;
    };
    uint32_t own = 0;
    for (int e = 0; e < each; ++e)
        if (b0 + e < p.batch) own = __builtin_elementwise_add_sat(own, (uint32_t)given(b0 + e));
    uint32_t upto = own;
    auto add = [&](uint32_t v) { upto = __builtin_elementwise_add_sat(upto, v); };
    add(dpp_move_u32<0x111, 0xf>(0, upto));
    add(dpp_move_u32<0x112, 0xf>(0, upto));
    add(dpp_move_u32<0x114, 0xf>(0, upto));
    add(dpp_move_u32<0x118, 0xf>(0, upto));
    add(dpp_move_u32<0x142, 0xa>(0, upto));
    add(dpp_move_u32<0x143, 0xc>(0, upto));
    if (lane == 63) s_wave[wave] = upto;
    uint32_t before = (uint32_t)__shfl_up((int)upto, 1, kWave), all = 0;
    if (lane == 0) before = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TRIM_THREADS / 64; ++w) {
        if (w < wave) before = __builtin_elementwise_add_sat(before, s_wave[w]);
        all = __builtin_elementwise_add_sat(all, s_wave[w]);
    }
    const int n_free = min(max(*p.n_free, 0), p.stack_size), room = p.stack_size - n_free;
    const int made = (int)min(all, (uint32_t)room);  // (the others are lost)
    for (int e = 0; e < each; ++e) {
        const int b = b0 + e;
        if (b >= p.batch) break;
        const int n = max(min(p.kv_lens[b], held), 0);
        s_start[b] = (int)min(before, (uint32_t)INT32_MAX);
        before = __builtin_elementwise_add_sat(before, (uint32_t)given(b));
        if (blockIdx.x == 0) {
            p.kv_out[b] = n > p.limit ? p.keep : n;
            p.evicted[b] = n > p.limit ? n - p.keep : 0;
        }
    }
    if (blockIdx.x == 0 && tid == 0) *p.n_free_out = n_free + made;
    __syncthreads();
    for (int i = blockIdx.x * TRIM_THREADS + tid; i < made; i += gridDim.x * TRIM_THREADS) {
        int b = 0;  // the last request that has no more than i pages before it
        for (int step = 1 << (31 - __builtin_clz(p.batch)); step > 0; step >>= 1) b = b + step < p.batch && s_start[b + step] <= i ? b + step : b;
        p.free_pages[n_free + i] = p.tables[(size_t)b * p.width + pages(p.keep) + (i - s_start[b])];
    }
}

}  // namespace

AGPU_EXPORT int32_t agpu_paged_evict(agpu_ctx *ctx, void *k_cache, void *v_cache, int64_t k_page_stride, int64_t v_page_stride, float *weights,
                                     int64_t weights_page_stride, const int32_t *block_tables, const int32_t *kv_lens, int32_t batch,
                                     int32_t n_kv_heads, int32_t n_pages, int32_t page_size, int32_t table_width, int32_t limit, int32_t keep,
                                     int32_t recent, int32_t sinks, int32_t d_head, int32_t cache_type) {
    AGPU_REQUIRE_CTX(ctx);
    paged::Refusal no = paged::refuse_cache((uintptr_t)k_cache, (uintptr_t)v_cache, k_page_stride, v_page_stride, n_kv_heads, n_pages, page_size, d_head, cache_type);
    if (no.code == AGPU_OK) no = paged::refuse_weights((uintptr_t)weights, weights_page_stride, n_kv_heads, n_pages, page_size);
    if (no.code == AGPU_OK) no = paged::refuse_budget(batch, table_width, page_size, limit, keep, recent, sinks);
    if (no.code == AGPU_OK) no = paged::refuse_evict(batch, n_kv_heads, table_width, page_size);
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_evict: %s", no.why);
    const int held = table_width * page_size;
    if (batch == 0 || held <= limit) return AGPU_OK;
    if (!k_cache || !v_cache || !weights || !block_tables || !kv_lens) return agpu_fail(ctx, AGPU_ERR_NULL_POINTER, "paged_evict: null pointer");
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    const int bytes = paged::cache_element_bytes(cache_type);
    const EvictArgs p = {static_cast<char *>(k_cache), static_cast<char *>(v_cache), k_page_stride * bytes, v_page_stride * bytes, weights, weights_page_stride, block_tables, kv_lens,
                         n_kv_heads, n_pages, table_width, held, limit, keep, recent, sinks, PageDiv::of(page_size)};
    const size_t lds = (size_t)((held + 63) / 64) * sizeof(uint64_t);
    auto go = [&](auto kernel) -> int32_t {
        if (lds > 32768) {  // (more than a launch gets unasked, together with what the kernel declares)
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return agpu_hip(ctx, e, "hipFuncSetAttribute");
        }
        hipLaunchKernelGGL(kernel, dim3((unsigned)(batch * n_kv_heads)), dim3(kEvictThreads), lds, ctx->stream, p);
        return AGPU_LAUNCH_CHECK(ctx, "paged_evict_kernel");
    };
    return cache_type == AGPU_CACHE_F32 ? go(paged_evict_kernel<16>) : go(paged_evict_kernel<8>);
}

AGPU_EXPORT int32_t agpu_paged_trim(agpu_ctx *ctx, const int32_t *kv_lens, const int32_t *block_tables, int32_t *free_pages, const int32_t *n_free, int32_t *kv_lens_out,
                                    int32_t *evicted, int32_t *n_free_out, int32_t batch, int32_t table_width, int32_t stack_size, int32_t page_size, int32_t limit,
                                    int32_t keep) {
    AGPU_REQUIRE_CTX(ctx);
    paged::Refusal no = paged::refuse_budget(batch, table_width, page_size, limit, keep, 0, 0);
    if (no.code == AGPU_OK) no = paged::refuse_plan(batch, table_width, stack_size, page_size, 0);
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_trim: %s", no.why);
    if ((batch > 0 && (!kv_lens || !kv_lens_out || !evicted || (!block_tables && table_width > 0))) || (!free_pages && stack_size > 0) || !n_free || !n_free_out)
        return agpu_fail(ctx, AGPU_ERR_NULL_POINTER, "paged_trim: null pointer");
    if ((batch > 0 && (kv_lens_out == kv_lens || evicted == kv_lens)) || n_free_out == n_free)
        return agpu_fail(ctx, AGPU_ERR_UNSUPPORTED, "paged_trim: the outputs do not overlap the inputs");
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    const TrimArgs p = {kv_lens, block_tables, n_free, free_pages, kv_lens_out, evicted, n_free_out, batch, table_width, stack_size, limit, keep, PageDiv::of(page_size)};
    // as many workgroups as there could be pages for, and as find a CU each
    const int64_t most = std::min<int64_t>(stack_size, (int64_t)batch * std::max(0, table_width - keep / page_size));
    const int groups = (int)std::max<int64_t>(1, std::min<int64_t>((most + 4 * TRIM_THREADS - 1) / (4 * TRIM_THREADS), ctx->num_cus));
    hipLaunchKernelGGL(paged_trim_kernel, dim3(groups), dim3(TRIM_THREADS), (batch + 1) * sizeof(int), ctx->stream, p);
    return AGPU_LAUNCH_CHECK(ctx, "paged_trim_kernel");
}
