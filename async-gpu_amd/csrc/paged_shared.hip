// Attention of requests that begin alike, d_head = 64: o = softmax(q k / 8) v over the keys of a prefix, which lies in the cache once, and of each request's own pages behind
// it.  The rows of all requests behind a prefix are rows of one product with its keys: paged_prefix_kernel takes them in tiles of 128 on the matrix cores and leaves o, m and
// l (sum of weights 2^(s - m), and their sum) of each row, in runs of keys; the kernels of paged_attention.hip then attend over the requests' own pages and join that in.
#include "paged_kernels.h"

namespace {

// The requests' rows, counted by prefix, and the places of a tile's rows.
struct PrefixShared {
    int rows[paged::kMaxPrefixes];
    int token[TILE_ROWS], pos[TILE_ROWS];
    int wave_rows[4];
};

// The rows that the call has of request b: how many, and the first.
__device__ __forceinline__ int rows_of(const PagedAttn &p, int b, int &start) {
    start = p.query_start ? p.query_start[b] : b;
    const int end = min(p.query_start ? p.query_start[b + 1] : b + 1, p.tokens);
    return start >= 0 && end > start ? end - start : 0;
}

// p.tables, p.width and p.held are the prefixes'.
template <class T>
__global__ __launch_bounds__(256, 2) void paged_prefix_kernel(const PagedAttn p, Runs cut, int cus, const More<PREFIX> more) {
    __shared__ TileShared<T> tile;
    __shared__ Units list;
    __shared__ PrefixShared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = p.group.size;
    if (tid < paged::kMaxPrefixes) s.rows[tid] = 0;
    __syncthreads();
    for (int b = tid; b < p.batch; b += 256) {
        const int g = more.of[b];
        int start;
        const int n = (unsigned)g < (unsigned)more.n_prefix ? rows_of(p, b, start) : 0;
        if (n > 0) atomicAdd(&s.rows[g], n);
    }
    __syncthreads();
    if (tid < paged::kMaxPrefixes) s.rows[tid] = min(s.rows[tid], p.tokens);
    __syncthreads();
    int tiles[4], keys[4], longest = 0;
    float work = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        tiles[j] = keys[j] = 0;
        if (64 * j >= more.n_prefix) continue;  // uniform
        const int g = 64 * j + lane;
        if (g < more.n_prefix) {
            keys[j] = more.len(g);
            tiles[j] = keys[j] > 0 ? (s.rows[g] * group + TILE_ROWS - 1) / TILE_ROWS : 0;
        }
        work += (float)tiles[j] * (float)keys[j];
        longest = max(longest, keys[j]);
    }
    cut.run = paged::run_for(wave_sum(work) * p.n_kv, 2.0f * cus, 128, (int)wave_minmax_u32<true>((unsigned)longest), cut.most);
    if (blockIdx.x == 0 && tid == 0) *more.run = cut.run;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (64 * j < more.n_prefix) tiles[j] *= paged::runs_of(keys[j], cut.run, cut.most).runs * p.n_kv;
    const int all = list.number(tiles, more.n_prefix, lane);
    for (int unit = blockIdx.x; unit < all; unit += gridDim.x) {
        __syncthreads();  // the numbers, and what the last unit left
        int at = unit;
        const int g = list.entry(at, lane), rows = s.rows[g] * group, n = (rows + TILE_ROWS - 1) / TILE_ROWS;
        const int runs = paged::runs_of(more.len(g), cut.run, cut.most).runs;
        const int place = at / n, first_row = (at - place * n) * TILE_ROWS;
        const int h = place / runs, run = place - h * runs;
        // which tokens the tile's rows are of: the prefix's tokens in the order of the requests
        const int first = p.group.page(first_row), last = p.group.page(min(first_row + TILE_ROWS, rows) - 1);
        int before = 0;
        for (int b0 = 0; b0 < p.batch && before <= last; b0 += 256) {
            const int b = b0 + tid;
            int start = 0, count = 0, pos = 0;
            if (b < p.batch && more.of[b] == g) {
                count = rows_of(p, b, start);
                pos = more.len(g) + min(max(p.kv_lens[b], 0), (int)paged::kMaxPositions) - (p.query_start ? p.query_start[b + 1] - start : 1);
            }
            const int upto = wave_running_sum(count);
            if (lane == 63) s.wave_rows[wave] = upto;
            __syncthreads();
            int at = before + upto - count;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (w < wave) at += s.wave_rows[w];
                before += s.wave_rows[w];
            }
            for (int i = max(first - at, 0); i < count && at + i <= last; ++i) {
                s.token[at + i - first] = start + i;
                s.pos[at + i - first] = pos + i;
            }
            __syncthreads();
        }
        tile_run<T>(p, more, tile, cut, g, TileOf<PREFIX>{s.token, s.pos, first, s.rows[g], p.group}, h, first_row, run, 0);
    }
}

}  // namespace

AGPU_EXPORT int32_t agpu_paged_attention_shared(agpu_ctx *ctx, const float *q, int64_t q_token_stride, int64_t q_head_stride, const void *k_cache,
                                                const void *v_cache, int64_t k_page_stride, int64_t v_page_stride, const int32_t *prefix_tables,
                                                const int32_t *prefix_lens, const int32_t *prefix_of, const int32_t *block_tables,
                                                const int32_t *kv_lens, const int32_t *query_start, float *o, int32_t tokens, int32_t batch,
                                                int32_t n_heads, int32_t n_kv_heads, int32_t n_pages, int32_t page_size, int32_t n_prefix,
                                                int32_t prefix_width, int32_t table_width, int32_t window, int32_t sinks, int32_t d_head,
                                                int32_t cache_type) {
    AGPU_REQUIRE_CTX(ctx);
    const paged::Refusal cache =
        paged::refuse_cache((uintptr_t)k_cache, (uintptr_t)v_cache, k_page_stride, v_page_stride, n_kv_heads, n_pages, page_size, d_head, cache_type);
    paged::Refusal no = paged::refuse_attention(tokens, batch, n_heads, n_kv_heads, table_width, page_size, window, sinks, query_start != nullptr);
    if (no.code == AGPU_OK) no = cache;
    if (no.code == AGPU_OK) no = paged::refuse_shared(n_prefix, prefix_width, table_width, page_size);
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_attention_shared: %s", no.why);
    if (tokens == 0 || batch == 0) return AGPU_OK;
    const bool any = n_prefix > 0 && prefix_width > 0;
    if (!q || !k_cache || !v_cache || !kv_lens || !o || (!block_tables && table_width > 0) || !prefix_of || (any && (!prefix_tables || !prefix_lens)))
        return agpu_fail(ctx, AGPU_ERR_NULL_POINTER, "paged_attention_shared: null pointer");
    if (!any)
        return agpu_paged_attention(ctx, q, q_token_stride, q_head_stride, k_cache, v_cache, k_page_stride, v_page_stride, block_tables, kv_lens, query_start, o, tokens, batch,
                                    n_heads, n_kv_heads, n_pages, page_size, table_width, window, sinks, d_head, cache_type);
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    const PagedAttn p = paged_attn(q, q_token_stride, q_head_stride, k_cache, v_cache, k_page_stride, v_page_stride, block_tables, kv_lens, query_start, o, tokens, batch, n_heads,
                             n_kv_heads, n_pages, page_size, table_width, window, sinks, ctx->strict_sync);
    // Scratch: the length of a run, (m, l) of the prefix's runs and o of all but the first, half of it at most; then the partial results over own pages.
    const paged::PrefixRuns room = paged::prefix_runs((int64_t)tokens * n_heads, (int64_t)prefix_width * page_size, ctx->ws_bytes);
    if (room.most == 0) return agpu_fail(ctx, AGPU_ERR_WORKSPACE, "paged_attention_shared: %d rows of %d heads need a larger scratch", tokens, n_heads);
    More<PREFIX> pre{};
    pre.tables = prefix_tables; pre.lens = prefix_lens; pre.of = prefix_of; pre.n_prefix = n_prefix; pre.width = prefix_width; pre.held = prefix_width * page_size;
    pre.run = reinterpret_cast<int *>(ctx->workspace);
    pre.ml = reinterpret_cast<float2 *>(ctx->workspace + 256);
    pre.rest = reinterpret_cast<float *>(ctx->workspace + room.rest);
    pre.most = room.most;
    const int64_t tiles = ((int64_t)tokens * p.group.size / TILE_ROWS + n_prefix) * n_kv_heads;
    PagedAttn front = p;
    front.tables = prefix_tables; front.width = prefix_width; front.held = pre.held;
    return of_type(cache_type, [&](auto type) {
        using T = decltype(type);
        const Runs cut = {128, room.most, nullptr, 0, nullptr};
        hipLaunchKernelGGL((paged_prefix_kernel<T>), dim3((unsigned)std::min<int64_t>(tiles * room.most, 2 * ctx->num_cus)), dim3(256), 0, ctx->stream, front, cut, ctx->num_cus, pre);
        const int32_t rc = AGPU_LAUNCH_CHECK(ctx, "paged_prefix_kernel");
        if (rc != AGPU_OK) return rc;
        return attention_go<T, SHARED>(ctx, p, paged::longest_row(p.held, window, sinks), static_cast<const More<SHARED> &>(pre), ctx->workspace + room.bytes, ctx->ws_bytes - room.bytes);
    });
}
