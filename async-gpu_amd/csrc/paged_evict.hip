// A KV cache cut down to a budget: which places of a request keep their keys, and the pages behind them.
//
// paged_evict_kernel, a workgroup a request and K/V head: weights as integers in the order of the floats, those that stay found by histograms of 11 bits from the top down until what
// is not decided is few, or all equal, and in the order of the places then.  What stays keeps its place, except where that is behind what is kept: it moves into the place of an
// evicted one, the first to the first.  So no more is moved than has to be (of 2200 keys cut down to 2000, 200), sources and targets never overlap, and nothing waits for the order of moves.
// What bounds it: 8 requests of 1000 to 1200 keys, 12 heads, fp32, 10.4 us, a chain: 1.6 to the first weights, 1.4 a histogram, 2 who stays, 1.4 the lists, 2 the moves.  64 requests
// of up to 4096 keys, 25 heads, bf16, cut to 2000: 58 us where it is done again and 170 MB move, 2.9 TB/s; the first time (3 times as much) the bytes.  Found bit by bit, two a step
// with a count each, the last weight that stays took 4 to 11 us in place of 3.
#include "agpu_internal.h"
#include "paged.h"

#include <algorithm>

namespace {

using paged::HolesMoves;
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
constexpr int kBins = 2048, kClose = 64;  // how many are told apart one by one

// Larger for larger weights; zeros of both signs are equal; no number is less than all numbers, and a page outside the cache (0) less than that.
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    return w != w ? 1u : (u >> 31) ? ~u : u | 0x80000000u;
}

struct EvictShared {
    int bins[kBins];
    uint32_t wave_sums[kEvictWaves];
    int found[3];  // the bin that what stays ends in, how many are above it, and in it
    int n_close;
    uint32_t close_key[kClose];
    int close_at[kClose];
    int ties[kEvictEach * kEvictWaves];  // of each 64 positions of a block
    HolesMoves before[kEvictThreads];    // in front of each 64 positions of 64 * 512
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
    auto beyond = [&](int block, int e) { return block * BLOCK + e * kEvictThreads >= n; };  // (uniform: nothing there)
    auto middle = [&](int i) { return i >= p.sinks && i < n - p.recent; };
    uint32_t key[kEvictEach];
    auto load = [&](int block) __attribute__((always_inline)) {
        int page[kEvictEach], slot[kEvictEach];
#pragma unroll
        for (int e = 0; e < kEvictEach; ++e) {
            const int i = block * BLOCK + e * kEvictThreads + tid;
            slot[e] = -1;
            if (beyond(block, e)) continue;
            if (middle(i)) slot[e] = slot_of(i, page[e]);
        }
#pragma unroll
        for (int e = 0; e < kEvictEach; ++e) key[e] = slot[e] >= 0 ? order_of(p.weights[page[e] * p.w_page + slot[e]]) : 0;
    };
    load(0);
    // The weight that what stays ends in, 11, 11 and 10 bits at a time: keys of the right upper bits (`least` >> upto) are counted by the next ones, until those that are not decided
    // are few, or all stay.  (The first 11 bits are a quarter of an octave.)
    uint32_t least = 0;
    int upto = 32, left = need, close = n - p.sinks - p.recent;  // of the `close` keys that agree with `least` down to bit `upto`, `left` stay
    while (left > 0 && left < close && close > kClose && upto > 0) {
        const int bits = upto > 10 ? 11 : 10, shift = upto - bits, bins = 1 << bits;
        for (int i = tid; i < bins; i += kEvictThreads) s.bins[i] = 0;
        __syncthreads();
        for (int block = 0; block < blocks; ++block) {
            if (blocks > 1) load(block);
#pragma unroll
            for (int e = 0; e < kEvictEach; ++e) {
                if (beyond(block, e)) break;
                const bool in = middle(block * BLOCK + e * kEvictThreads + tid) && (upto == 32 || key[e] >> (upto & 31) == least >> (upto & 31));
                if (in) atomicAdd(&s.bins[key[e] >> shift & (bins - 1)], 1);
            }
        }
        __syncthreads();
        // from the top down: a thread has a few bins
        const int each = bins / kEvictThreads, first = bins - 1 - each * tid;
        int own = 0;
        for (int i = 0; i < each; ++i) own += s.bins[first - i];
        const int sum = wave_running_sum(own);
        if (lane == 63) s.wave_sums[wave] = (uint32_t)sum;
        __syncthreads();
        int above = sum - own;
#pragma unroll
        for (int w = 0; w < kEvictWaves; ++w) above += w < wave ? (int)s.wave_sums[w] : 0;
        if (above < left && above + own >= left) {  // (one thread's)
            int i = 0;
            while (above + s.bins[first - i] < left) above += s.bins[first - i++];
            s.found[0] = first - i;
            s.found[1] = above;
            s.found[2] = s.bins[first - i];
        }
        __syncthreads();
        least |= (uint32_t)s.found[0] << shift;
        left -= s.found[1];
        close = s.found[2];
        upto = shift;
    }
    // Who stays, a bit a position: above all that are close; of these none, all, the first of equal ones, or what comes out one by one.
    const bool all_close = left > 0 && left >= close, one_by_one = left > 0 && !all_close && upto > 0, equal = left > 0 && !all_close && upto == 0;
    if (tid == 0) s.n_close = 0;
    if (tid < kClose) s.close_key[tid] = s.close_at[tid] = 0;
    int ties = left;
    __syncthreads();
    for (int block = 0; block < blocks; ++block) {
        if (blocks > 1) load(block);
        int before = 0, all = 0;
        uint64_t same[kEvictEach];
        if (equal) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kEvictEach; ++e) {
                same[e] = __ballot(middle(block * BLOCK + e * kEvictThreads + tid) && key[e] == least);
                if (lane == 0) s.ties[e * kEvictWaves + wave] = __popcll(same[e]);
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
            if (beyond(block, e)) break;
            const int i = block * BLOCK + e * kEvictThreads + tid;
            const bool inside = middle(i), near = inside && (upto == 32 || key[e] >> (upto & 31) == least >> (upto & 31));
            bool stay = i < n && (!inside || (!near && key[e] > least));
            if (near && all_close) stay = true;
            if (near && equal) stay = __builtin_amdgcn_readlane(before, e * kEvictWaves + __builtin_amdgcn_readfirstlane(wave)) + bits_below(same[e]) < ties;
            if (near && one_by_one) {
                const int at = atomicAdd(&s.n_close, 1);  // (in any order: what comes out does not depend on it)
                if (at < kClose) {                        // (more only where weights change meanwhile, on a page that another request has too)
                    s.close_key[at] = key[e];
                    s.close_at[at] = i;
                }
            }
            const uint64_t word = __ballot(stay);
            const int chunk = (block * kEvictEach + e) * kEvictWaves + wave;
            if (lane == 0 && chunk < chunks) stays[chunk] = word;
        }
        ties -= all;
    }
    __syncthreads();
    if (one_by_one) {
        static_assert(8 * kClose == kEvictThreads, "");
        const int own = min(tid >> 3, close - 1), at = s.close_at[own];  // eight threads for each
        const uint32_t mine = s.close_key[own];
        int before = 0;
#pragma unroll
        for (int e = 0; e < kClose / 8; ++e) {
            const int i = 8 * e + (tid & 7), k = min(i, close - 1);
            before += i < close && (s.close_key[k] > mine || (s.close_key[k] == mine && s.close_at[k] < at));
        }
        before += (int)dpp_move_u32<0xb1, 0xf>(0, before);   // quad_perm [1,0,3,2]
        before += (int)dpp_move_u32<0x4e, 0xf>(0, before);   // quad_perm [2,3,0,1]
        before += (int)dpp_move_u32<0x141, 0xf>(0, before);  // row_half_mirror
        if ((tid & 7) == 0 && tid >> 3 < close && before < left) atomicOr(reinterpret_cast<unsigned int *>(stays) + (at >> 5), 1u << (at & 31));
        __syncthreads();
    }
    // Of 64 positions those that are evicted and get another one's key, or those that move.
    auto word = [&](bool hole, int chunk) {
        const uint64_t kept = first_bits(p.keep - 64 * chunk), stay = stays[chunk];
        return hole ? ~stay & kept : stay & ~kept;
    };
    // Numbers done .. done + kEvictListed - 1 of the ones or the other, or both, of 64 * 512 positions at a time, beginning with the group in which the first of them is.
    struct Cursor {
        int group, before;  // and how many there are before that group
    };
    Cursor hole = {0, 0}, move = {p.keep / (64 * kEvictThreads), 0};
    int moves = 1 << 30;  // (known when all positions have been gone through)
    auto list = [&](bool holes, bool movers, int done) __attribute__((always_inline)) {
        for (;;) {
            const int group = holes ? hole.group : move.group, chunk = group * kEvictThreads + tid;
            const uint32_t own = chunk < chunks ? HolesMoves::of(__popcll(word(true, chunk)), __popcll(word(false, chunk))).both : 0;
            const uint32_t sum = (uint32_t)wave_running_sum((int)own);  // (of a wave 2^28 at most)
            if (lane == 63) s.wave_sums[wave] = sum;
            __syncthreads();
            uint32_t before = sum - own;
            HolesMoves all = {0};
#pragma unroll
            for (int w = 0; w < kEvictWaves; ++w) {
                if (w < wave) before += s.wave_sums[w];
                all.both += s.wave_sums[w];
            }
            s.before[tid] = {before};
            __syncthreads();
            const int hole_base = hole.before - done, move_base = move.before - done, all_holes = all.holes(), all_moves = all.moves();
            for (int c = wave; c < kEvictThreads && group * kEvictThreads + c < chunks; c += kEvictWaves) {
                const int at = group * kEvictThreads + c;
                const HolesMoves front = s.before[c];
                auto note = [&](bool which, int rank, int *out) {
                    const uint64_t bits = word(which, at);
                    rank += bits_below(bits);
                    if ((bits >> lane & 1) && rank >= 0 && rank < kEvictListed) out[rank] = 64 * at + lane;
                };
                if (holes) note(true, hole_base + front.holes(), s.to);
                if (movers) note(false, move_base + front.moves(), s.from);
            }
            __syncthreads();
            const bool end = (group + 1) * kEvictThreads >= chunks;
            if (movers && end) moves = move.before + all_moves;
            const bool more_holes = holes && !end && hole.before + all_holes < done + kEvictListed, more_moves = movers && !end && move.before + all_moves < done + kEvictListed;
            if (more_holes) hole = {group + 1, hole.before + all_holes};
            if (more_moves) move = {group + 1, move.before + all_moves};
            if (!more_holes && !more_moves) return;
            holes = more_holes;
            movers = more_moves;
        }
    };
    for (int done = 0; done < moves; done += kEvictListed) {
        if (hole.group == move.group) {
            list(true, true, done);
        } else {
            list(false, true, done);
            list(true, false, done);
        }
        const int now = min(moves - done, kEvictListed);
        constexpr int ROUNDS = 4;
        typedef uint32_t Piece __attribute__((ext_vector_type(4)));
        for (int base = 0; base < now * ROW; base += ROUNDS * kEvictThreads) {
            Piece kx[ROUNDS], vx[ROUNDS];
            float w[ROUNDS];
            int from_page[ROUNDS], to_page[ROUNDS], from[ROUNDS], to[ROUNDS];
            const int piece = tid % ROW;
            bool ok[ROUNDS];
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r) {
                const int i = base + r * kEvictThreads + tid, m = min(i / ROW, now - 1);
                // (Every position that moves has one to go to, but where weights changed meanwhile; whatever is in the lists then, it is kept to the request's own positions.)
                from[r] = slot_of((int)min((uint32_t)s.from[m], (uint32_t)n - 1), from_page[r]);
                to[r] = slot_of((int)min((uint32_t)s.to[m], (uint32_t)n - 1), to_page[r]);
                ok[r] = i < now * ROW && from[r] >= 0 && to[r] >= 0;
                if (!ok[r]) from[r] = from_page[r] = 0;  // (loaded all the same, so that all loads are on their way together)
            }
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r) {
                const long long at = ((long long)from[r] * ROW + piece) * 16;
                kx[r] = *reinterpret_cast<const Piece *>(p.k + from_page[r] * p.k_page + at);
                vx[r] = *reinterpret_cast<const Piece *>(p.v + from_page[r] * p.v_page + at);
                w[r] = p.weights[from_page[r] * p.w_page + from[r]];
            }
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r)
                if (ok[r]) {
                    const long long at = ((long long)to[r] * ROW + piece) * 16;
                    *reinterpret_cast<Piece *>(p.k + to_page[r] * p.k_page + at) = kx[r];
                    *reinterpret_cast<Piece *>(p.v + to_page[r] * p.v_page + at) = vx[r];
                    if (piece == 0) p.weights[to_page[r] * p.w_page + to[r]] = w[r];
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

// Every workgroup adds up the pages of all requests for itself, then they share the stack's new entries.  8 requests 2.2 us, 512 that give 38000 pages back 4.9.
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
    const int bytes = paged::cache_element_bytes(cache_type);
    const paged::Pieces k = paged::cache_pages(k_cache, k_page_stride, n_kv_heads, n_pages, page_size, bytes), v = paged::cache_pages(v_cache, v_page_stride, n_kv_heads, n_pages, page_size, bytes);
    no = paged::refuse_evicted_memory(k, v, paged::weight_pages(weights, weights_page_stride, n_kv_heads, n_pages, page_size));
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_evict: %s", no.why);
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
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
    using paged::Pieces;
    constexpr int64_t kInt = sizeof(int32_t);
    const Pieces lens = Pieces::one(kv_lens, batch * kInt), tables = Pieces::one(block_tables, (int64_t)batch * table_width * kInt), count = Pieces::one(n_free, kInt);
    const Pieces out[4] = {Pieces::one(kv_lens_out, batch * kInt), Pieces::one(evicted, batch * kInt), Pieces::one(n_free_out, kInt), Pieces::one(free_pages, stack_size * kInt)};
    for (int i = 0; i < 4 && no.code == AGPU_OK; ++i) {
        no = paged::refuse_shared_memory(out[i], {lens, tables, count}, "the outputs do not overlap the inputs");
        for (int j = 0; j < i && no.code == AGPU_OK; ++j) no = paged::refuse_shared_memory(out[i], {out[j]}, "the outputs do not overlap");
    }
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_trim: %s", no.why);
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    const TrimArgs p = {kv_lens, block_tables, n_free, free_pages, kv_lens_out, evicted, n_free_out, batch, table_width, stack_size, limit, keep, PageDiv::of(page_size)};
    // as many workgroups as there could be pages for, and as find a CU each
    const int64_t most = std::min<int64_t>(stack_size, (int64_t)batch * std::max(0, table_width - keep / page_size));
    const int groups = (int)std::max<int64_t>(1, std::min<int64_t>((most + 4 * TRIM_THREADS - 1) / (4 * TRIM_THREADS), ctx->num_cus));
    hipLaunchKernelGGL(paged_trim_kernel, dim3(groups), dim3(TRIM_THREADS), (batch + 1) * sizeof(int), ctx->stream, p);
    return AGPU_LAUNCH_CHECK(ctx, "paged_trim_kernel");
}
