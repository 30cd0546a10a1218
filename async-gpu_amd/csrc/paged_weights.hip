// Attention that adds up the weight that each key was given (over the rows of a call and the query heads of a K/V head), d_head = 64: the kernels of paged_attention.hip, and
//   one row a request   its scores stay in scratch (4 bytes a key and query head beside 128 to 512 of K and V).  The workgroup that joins the row's runs, which knows m and l by then,
//                       turns them into weights, or, where there are many keys, a launch of its own: 64 tokens of 1 to 4096 keys, 32 heads over 8, f16, 41 us (attention alone 28).
//   more                m and 1 / l of the rows stay in scratch, and paged_weights_kernel forms their scores once more on the matrix cores, a wave's 32 keys in registers
//                       against all rows that see them, 64 at a time: a key's sum is one wave's, in the order of the rows.  4 chunks of 512 rows over 2048 keys, 16 heads, fp32, 53 us
//                       beside 102 of attention: matrix instructions 33 % and vector instructions 38 % of the SIMDs' cycles, which overlap little; matrix instructions alone would take 32.
//                       Half of what it was to begin with went to conflicts between LDS banks (66 us).
#include "paged_kernels.h"

namespace {

// ---- what each key was given, by several rows of a request ------------------------------------------

// The rows of a step of twice 32 in LDS, as operands, double buffered.
template <class T>
struct RowsShared {
    uint4 q[2][2][Tiles<T>::QP][kFrag];  // [d step of 16][half][row ^ 2 (twice the step + half): what is written at a time lies in all banks]
    float unit[2][2][32];                // f16: of the scores
};

// Sum over the 32 lanes of a half wave, in each of them.
__device__ __forceinline__ float half_wave_sum(float v) {
    v = row16_sum(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The 128 keys from number `first_key` on of those that the rows of request b see, for K/V head h.  n: rows of the request, `there` of them in the call.
template <class T>
__device__ __forceinline__ void weigh_keys(const PagedAttn &p, const More<WEIGHTS> &more, RowsShared<T> &s, int b, int start, int n, int there, int h, int first_key) {
    constexpr int KP = Tiles<T>::KP, QP = Tiles<T>::QP, kBytes = 16 / T::EL;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, h2 = lane >> 5, group = p.group.size;
    const int kv_len = max(p.kv_lens[b], 0), pos_first = kv_len - n;
    const paged::TileKeys keys = paged::tile_keys(pos_first, kv_len - 1, p.held, p.window, p.sinks);
    const int stay = max(p.sinks - keys.gap, keys.first);  // numbers below it are seen whatever the window
    // this wave's keys
    const int v0 = first_key + 32 * wave, v = v0 + c, j = keys.key(v);
    const char *row = static_cast<const char *>(p.k);
    float *to = more.weights;
    bool real = false;
    if (v < keys.count) {
        const int at = p.div.page(j), place = j - at * p.div.size, page = p.tables[(size_t)b * p.width + at];
        real = (unsigned)page < (unsigned)p.n_pages;
        if (real) {
            row += (page * p.k_page + (long long)(h * p.div.size + place) * DH) * kBytes;
            to += page * more.page + (long long)h * p.div.size + place;
        }
    }
    const uint32_t held = (uint32_t)__ballot(real);  // (both halves have the same keys)
    const float old = real && j < pos_first ? *to : 0.0f;
    uint4 k[4][KP];
    bool odd = false;
    {
        Staged<T> x[4];
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) {
            x[ds].row(row + (16 * ds + 8 * h2) * kBytes);
            if (!real) x[ds].clear();
            if (__any(x[ds].odd())) odd |= x[ds].clean() != 0;
            x[ds].pieces(k[ds]);
        }
    }
    uint32_t odd_k = (uint32_t)__ballot(odd) | (uint32_t)(__ballot(odd) >> 32);

    // Rows from the first that sees a key of the workgroup's to the last that does, in steps of 64.
    const int last_key = min(first_key + 128, keys.count) - 1;
    const int from = min(max(keys.key(first_key) - pos_first, 0), there);
    int upto = there;
    if (p.window > 0 && first_key >= stay) upto = (int)max(min((long long)there, (long long)keys.key(last_key) + p.window - pos_first), 0ll);
    const int row_from = from * group & ~31, row_upto = upto * group;
    const int steps = row_upto > row_from ? (row_upto - row_from + 63) / 64 : 0;
    // what this thread fetches of a step: eight elements of two of its rows, and what weights of its lane's rows are in units of and divided by
    const int own = tid >> 3, part = tid & 7;
    float4 qa[2], qd[2];
    float2 next_stats[2];
    auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int own_r = min(row_from + 64 * i + 32 * u + c, row_upto - 1), own_token = p.group.page(own_r);
            next_stats[u] = more.stats[(size_t)(start + own_token) * p.n_heads + h * group + (own_r - own_token * group)];
            const int r = min(row_from + 64 * i + 32 * u + own, row_upto - 1), token = p.group.page(r), head = h * group + (r - token * group);
            const float *from = p.q + (size_t)(start + token) * p.q_row + (size_t)head * p.q_head + 8 * part;
            qa[u] = load4(from);
            qd[u] = load4(from + 4);
        }
    };
    if (steps > 0) fetch(0);
    float acc[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
    const int v_last = v0 + 31;
    for (int i = 0; i < steps; ++i) {
        const int buf = i & 1;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float x[8] = {qa[u].x, qa[u].y, qa[u].z, qa[u].w, qd[u].x, qd[u].y, qd[u].z, qd[u].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= kQueryScale;
            if (QP == 2) {  // as in a tile of rows: into 2^14 .. 2^15
                float most = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
                most = fmaxf(most, dpp_move<0xb1, 0xf>(most, most));
                most = fmaxf(most, dpp_move<0x4e, 0xf>(most, most));
                most = fmaxf(most, dpp_move<0x141, 0xf>(most, most));  // row_half_mirror: eight lanes have a row
                const int up = max(min(141 - (int)((__float_as_uint(most) >> 23) & 255u), 100), -112);
                const float by = __uint_as_float((uint32_t)(up + 127) << 23);
                if (part == 0) s.unit[buf][u][own] = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= by;
            }
            uint4 piece[QP];
            pieces_of(x, piece);
#pragma unroll
            for (int level = 0; level < QP; ++level) s.q[buf][u][level][part * 32 + (own ^ 2 * part)] = piece[level];
        }
        const float2 stats[2] = {next_stats[0], next_stats[1]};
        if (i + 1 < steps) fetch(i + 1);
        // this lane's rows of the step
        int pos[2], token[2], head[2];
        const int row0 = row_from + 64 * i;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = min(row0 + 32 * u + c, row_upto - 1);
            token[u] = p.group.page(r);
            head[u] = h * group + (r - token[u] * group);
            pos[u] = pos_first + token[u];
        }
        __syncthreads();
        floatx16 x[2] = {};
#pragma unroll
        for (int level = QP - 1; level >= 0; --level)
#pragma unroll
            for (int ds = 0; ds < 4; ++ds)
#pragma unroll
                for (int kp = KP - 1; kp >= 0; --kp)
                    if (level - kp >= 0 && level - kp < QP)
#pragma unroll
                        for (int u = 0; u < 2; ++u) x[u] = Tiles<T>::mfma(k[ds][kp], s.q[buf][u][level - kp][(2 * ds + h2) * 32 + (c ^ 2 * (2 * ds + h2))], x[u]);
        // only steps at the ends of what rows see hide anything (uniform)
        const int pos0 = pos_first + p.group.page(row0), pos1 = pos_first + p.group.page(min(row0 + 63, row_upto - 1));
        const bool whole = held == 0xffffffffu && row0 + 64 <= row_upto && v_last <= pos0 - keys.gap && (v0 > paged::row_keys(keys, pos1, p.window, p.sinks).low || v_last < stay);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (QP == 2) {
                const float unit = s.unit[buf][u][c];
#pragma unroll
                for (int e = 0; e < 16; ++e) x[u][e] *= unit;
            }
            if (__builtin_expect(odd_k != 0, 0)) {  // scores of keys with something infinite or no number, in fp32 (uniform)
                const float *q_row = p.q + (size_t)(start + token[u]) * p.q_row + (size_t)head[u] * p.q_head;
#pragma unroll 1
                for (int kk = 0; kk < 32; ++kk) {
                    if (!(odd_k >> kk & 1)) continue;
                    const char *key = reinterpret_cast<const char *>((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(uintptr_t)row, kk) |
                                                                     (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uintptr_t)row >> 32), kk) << 32);
                    float d = 0.0f;
#pragma unroll 1
                    for (int e = 0; e < 32; ++e) d = fmaf(q_row[32 * h2 + e] * kQueryScale, T::one(key, 32 * h2 + e), d);
                    d = sum_of_halves(d);
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[u][e] = 8 * (e >> 2) + 4 * h2 + (e & 3) == kk ? d : x[u][e];
                }
            }
            if (whole) {
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[e] = fmaf(__builtin_amdgcn_exp2f(x[u][e] - stats[u].x), stats[u].y, acc[e]);
                continue;
            }
            const paged::RowKeys see = paged::row_keys(keys, pos[u], p.window, p.sinks);
            auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; };  // bits 0 .. n - 1
            uint32_t seen = held & below(see.last + 1 - v0) & (~below(see.low + 1 - v0) | below(see.first - v0));
            if (row0 + 32 * u + c >= row_upto) seen = 0;
            seen >>= 4 * h2;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float w = __builtin_amdgcn_exp2f(x[u][e] - stats[u].x) * stats[u].y;
                acc[e] += seen >> (8 * (e >> 2) + (e & 3)) & 1 ? w : 0.0f;
            }
        }
    }
    float mine = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const float sum = half_wave_sum(acc[e]);
        // lane c of the half that has key c's sum
        mine = 8 * (e >> 2) + (e & 3) == (c & ~4) ? sum : mine;
    }
    if (real && (c >> 2 & 1) == h2) *to = old + mine;
}

// Keys number v0 .. of those that the only row of request b sees, four a thread, from the scores that attention has left.
constexpr int kScoredKeys = 1024;
__device__ __forceinline__ void add_scored(const PagedAttn &p, const More<WEIGHTS> &more, int b, int t, int h, int v0) {
    const int group = p.group.size, kv_len = max(p.kv_lens[b], 0), pos = kv_len - 1;
    const Visible vis = paged::visible(pos, kv_len, p.held, p.window, p.sinks);
    const int *table = p.tables + (size_t)b * p.width;
    const float2 *stats = more.stats + (size_t)t * p.n_heads + h * group;
    constexpr int EACH = kScoredKeys / 256;
    int place[EACH], page[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int v = v0 + 256 * k + (int)threadIdx.x, j = v < vis.count ? vis.key(v) : 0, at = p.div.page(j);
        place[k] = h * p.div.size + (j - at * p.div.size);
        page[k] = v < vis.count ? table[at] : -1;
    }
    float sum[EACH], old[EACH];
    const float *score[EACH];
    float *to[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const bool there = (unsigned)page[k] < (unsigned)p.n_pages;
        const size_t of = there ? page[k] : 0;
        score[k] = more.scores + more.score_at(p, b, h, min(v0 + 256 * k + (int)threadIdx.x, vis.count - 1), (int)of, place[k] - h * p.div.size);
        to[k] = more.weights + of * more.page + place[k];
        old[k] = *to[k];
        sum[k] = 0.0f;
        if (!there) to[k] = nullptr;
    }
    for (int g = 0; g < group; ++g) {
        const float2 row = stats[g];
#pragma unroll
        for (int k = 0; k < EACH; ++k) sum[k] += __builtin_amdgcn_exp2f(score[k][g] - row.x) * row.y;
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int v = v0 + 256 * k + (int)threadIdx.x;
        if (to[k] != nullptr) *to[k] = (vis.key(v) == pos ? 0.0f : old[k]) + sum[k];
    }
}

// Units: tiles of 128 keys of a request and K/V head, or of 1024 of one whose scores are there, 256 requests at a time.
template <class T>
__global__ __launch_bounds__(256, 2) void paged_weights_kernel(const PagedAttn p, const More<WEIGHTS> more) {
    __shared__ RowsShared<T> s;
    __shared__ Units list;
    __shared__ int starts[kListed], rows[kListed], in_call[kListed];
    const int lane = threadIdx.x & 63;
    int before = 0;  // units of the requests so far, modulo the grid
    for (int b0 = 0, skip = 0; b0 < p.batch;) {  // skip: tiles of each head that are done (where a request has more of them than are numbered at a time)
        __syncthreads();
        const int entries = min(p.batch - b0, kListed);
        int units[4];
        bool rest = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            units[j] = 0;
            if (64 * j >= entries) continue;  // uniform
            const int i = 64 * j + lane, b = b0 + i;
            if (i < entries) {
                const int start = p.query_start ? p.query_start[b] : b, end = p.query_start ? p.query_start[b + 1] : b + 1, kv_len = max(p.kv_lens[b], 0);
                const int there = min(end, p.tokens) - start;
                const bool scored = more.scored(end - start, p.group.size);
                if (start >= 0 && there > 0 && !(scored && more.few)) {
                    const int count = paged::tile_keys(kv_len - (end - start), kv_len - 1, p.held, p.window, p.sinks).count, each = scored ? kScoredKeys : 128;
                    const int tiles = max((count + each - 1) / each - skip, 0);
                    units[j] = min(tiles, more.at_once) * p.n_kv;
                    rest |= tiles > more.at_once;
                }
                starts[i] = start;
                rows[i] = end - start;
                in_call[i] = there;
            }
        }
        const int b_now = b0, skip_now = skip;
        if (__any(rest)) skip += more.at_once;  // uniform, and the same in every wave
        else b0 += kListed, skip = 0;
        if (!__any(units[0] + units[1] + units[2] + units[3] > 0)) continue;  // uniform: nobody here has several rows
        const int all = list.number(units, entries, lane);
        __syncthreads();
        const int grid = gridDim.x, first = (int)blockIdx.x >= before ? (int)blockIdx.x - before : (int)blockIdx.x - before + grid;
        for (int unit = first; unit < all; unit += grid) {
            int at = unit;
            const int i = list.entry(at, lane), h = at % p.n_kv, tile = skip_now + at / p.n_kv;
            if (more.scored(rows[i], p.group.size)) {
                add_scored(p, more, b_now + i, starts[i], h, kScoredKeys * tile);
            } else {
                weigh_keys<T>(p, more, s, b_now + i, starts[i], rows[i], in_call[i], h, 128 * tile);
                __syncthreads();
            }
        }
        before = (int)(((unsigned)before + (unsigned)all % (unsigned)grid) % (unsigned)grid);
    }
}

}  // namespace

AGPU_EXPORT int32_t agpu_paged_attention_weights(agpu_ctx *ctx, const float *q, int64_t q_token_stride, int64_t q_head_stride, const void *k_cache,
                                                 const void *v_cache, int64_t k_page_stride, int64_t v_page_stride, float *weights,
                                                 int64_t weights_page_stride, const int32_t *block_tables, const int32_t *kv_lens,
                                                 const int32_t *query_start, float *o, int32_t tokens, int32_t batch, int32_t n_heads,
                                                 int32_t n_kv_heads, int32_t n_pages, int32_t page_size, int32_t table_width, int32_t window,
                                                 int32_t sinks, int32_t d_head, int32_t cache_type) {
    AGPU_REQUIRE_CTX(ctx);
    const paged::Refusal cache =
        paged::refuse_cache((uintptr_t)k_cache, (uintptr_t)v_cache, k_page_stride, v_page_stride, n_kv_heads, n_pages, page_size, d_head, cache_type);
    paged::Refusal no = paged::refuse_attention(tokens, batch, n_heads, n_kv_heads, table_width, page_size, window, sinks, query_start != nullptr);
    if (no.code == AGPU_OK) no = cache;
    if (no.code == AGPU_OK) no = paged::refuse_weights((uintptr_t)weights, weights_page_stride, n_kv_heads, n_pages, page_size);
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_attention_weights: %s", no.why);
    if (tokens == 0 || batch == 0) return AGPU_OK;
    if (!q || !k_cache || !v_cache || !weights || !kv_lens || !o || (!block_tables && table_width > 0))
        return agpu_fail(ctx, AGPU_ERR_NULL_POINTER, "paged_attention_weights: null pointer");
    const int bytes = paged::cache_element_bytes(cache_type);
    no = paged::refuse_shared_memory(paged::weight_pages(weights, weights_page_stride, n_kv_heads, n_pages, page_size),
                                     {paged::cache_pages(k_cache, k_page_stride, n_kv_heads, n_pages, page_size, bytes), paged::cache_pages(v_cache, v_page_stride, n_kv_heads, n_pages, page_size, bytes),
                                      paged::Pieces::rows(q, tokens, n_heads, q_token_stride, q_head_stride), paged::Pieces::one(o, (int64_t)tokens * n_heads * DH * sizeof(float))},
                                     "the weights share memory with another argument");
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_attention_weights: %s", no.why);
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    const PagedAttn p = paged_attn(q, q_token_stride, q_head_stride, k_cache, v_cache, k_page_stride, v_page_stride, block_tables, kv_lens, query_start, o, tokens, batch, n_heads,
                                   n_kv_heads, n_pages, page_size, table_width, window, sinks, ctx->strict_sync);
    // Scores lie by requests, or by places of the cache, whichever are fewer (a large cache, or tables much wider than requests are long), as far as the arguments' sizes say: lengths are on
    // the device.  Without room for them they are formed again: 64 tokens of 1 to 4096 keys, 32 heads over 8, f16, 59 us, 41 with scores.
    const int64_t longest = paged::longest_row(p.held, window, sinks), by_place = (int64_t)n_pages * page_size, by_request = batch * longest;
    const paged::WeightsRoom room = paged::weights_room((int64_t)tokens * n_heads, std::min(by_place, by_request) * n_heads, n_heads / n_kv_heads, ctx->ws_bytes);
    if (room.bytes == 0) return agpu_fail(ctx, AGPU_ERR_WORKSPACE, "paged_attention_weights: %d rows of %d heads need a larger scratch", tokens, n_heads);
    More<WEIGHTS> more{};
    more.weights = weights; more.page = weights_page_stride;
    more.stats = reinterpret_cast<float2 *>(ctx->workspace);
    more.seen = by_request < by_place ? (int)longest : 0;
    more.scores = room.scores ? reinterpret_cast<float *>(ctx->workspace + room.scores) : nullptr;
    more.at_once = paged::weight_tiles(n_kv_heads);
    // The last workgroup at a token adds up its weights where other work goes on meanwhile (chunks beside tokens: 37 us, 39 with a launch for them), or where there is so little of it that
    // a launch more costs as much (12 heads of 777 keys: 10 us, and 4 for the launch where query_start leaves open whether there are chunks); 64 tokens of up to 4096 keys, 8 heads: 43 us that way, 40 with one.
    more.few = more.scores && (tokens > batch || (int64_t)tokens * n_kv_heads * std::min<int64_t>(longest, kScoredKeys) <= 64 * kScoredKeys);
    return of_type(cache_type, [&](auto type) {
        using T = decltype(type);
        int32_t rc = attention_go<T, WEIGHTS>(ctx, p, longest, more, ctx->workspace + room.bytes, ctx->ws_bytes - room.bytes);
        if (rc != AGPU_OK || (!query_start && more.few)) return rc;
        hipLaunchKernelGGL((paged_weights_kernel<T>), dim3(2 * ctx->num_cus), dim3(256), 0, ctx->stream, p, more);
        return AGPU_LAUNCH_CHECK(ctx, "paged_weights_kernel");
    });
}
