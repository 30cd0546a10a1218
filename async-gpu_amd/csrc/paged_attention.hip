// Attention over a KV cache in pages, d_head = 64: o = softmax(q k / 8) v for the rows of several requests, each over the keys of its own block table.
#include "agpu_internal.h"
#include "paged.h"

#include <algorithm>

namespace {

using paged::PageDiv;
using paged::Visible;

constexpr int DH = 64;

struct PagedAttn {
    const float *q;
    long long q_row, q_head;  // elements between tokens and between heads
    const void *k, *v;
    long long k_page, v_page;  // elements between pages
    const int *tables, *kv_lens, *query_start;
    float *o;  // [tokens][n_heads][64]
    int tokens, batch, n_heads, n_kv, n_pages, width, held, window, sinks;
    PageDiv div;
    int shortest_run, max_runs;  // of keys over workgroups
    float *partial;
    unsigned int *counters;
    int strict;
};

// Scores are in units of the binary logarithm: q is taken times log2(e) / 8.
constexpr float kQueryScale = 0.125f * 1.44269504088896340736f;

// ---- elements of the cache, 16 bytes a lane ----
struct F32 {
    static constexpr int EL = 4;
    static __device__ __forceinline__ void floats(const uint4 &x, float (&f)[4]) {
        f[0] = __uint_as_float(x.x); f[1] = __uint_as_float(x.y); f[2] = __uint_as_float(x.z); f[3] = __uint_as_float(x.w);
    }
};
struct BF16 {
    static constexpr int EL = 8;
    static __device__ __forceinline__ void floats(const uint4 &x, float (&f)[8]) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
struct F16 {
    static constexpr int EL = 8;
    static __device__ __forceinline__ void floats(const uint4 &x, float (&f)[8]) {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)w[i]);
            f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[i] >> 16));
        }
    }
};

// Sum over the LPK (8 or 16) lanes that share a key, in each of them.
template <int LPK>
__device__ __forceinline__ float sum_of_key(float v) {
    v += dpp_move<0xb1, 0xf>(0.0f, v);   // quad_perm [1,0,3,2]
    v += dpp_move<0x4e, 0xf>(0.0f, v);   // quad_perm [2,3,0,1]
    if (LPK == 8) return v + dpp_move<0x141, 0xf>(0.0f, v);  // row_half_mirror
    v += dpp_move<0x124, 0xf>(0.0f, v);  // row_ror:4
    return v + dpp_move<0x128, 0xf>(0.0f, v);  // row_ror:8
}
// op over the lanes LPK, 2 LPK, ... apart
template <int LPK, class F>
__device__ __forceinline__ float over_keys(float v, F op) {
    if (LPK == 8) v = op(v, dpp_move<0x128, 0xf>(0.0f, v));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// The request that token t belongs to (uniform; `batch`: behind the last one).
__device__ __forceinline__ int request_of(const int *query_start, int batch, int t, int lane) {
    if (!query_start) return t;
    if (t < batch && query_start[t] == t && query_start[t + 1] == t + 1) return t;  // one token each so far, as a rule
    int b = 0;
    for (int i = 0; i < batch; i += 64) b += __popcll(__ballot(i + lane < batch && query_start[i + lane + 1] <= t));
    return b;
}

// grid (tokens * n_kv * blocks, runs), 64 W threads: up to G query heads of a token that share a K/V head over a run of its keys.  LPK lanes share a key, 16 bytes each.
template <class T, int G, int W, int PASS>
__global__ __launch_bounds__(64 * W) void paged_tokens_kernel(const PagedAttn p) {
    constexpr int EL = T::EL, LPK = DH / EL, KEYS = 64 / LPK;
    __shared__ float s_o[W][G][DH], s_m[W][G], s_l[W][G];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = lane % LPK, own = lane / LPK;
    const int item = blockIdx.x, run = blockIdx.y;
    const int heads_all = p.n_heads / p.n_kv, blocks = (heads_all + G - 1) / G;  // (G is the power of two that covers them, up to 8)
    const int t = item / (p.n_kv * blocks), hb = item - t * p.n_kv * blocks, h = hb / blocks, g0 = (hb - h * blocks) * G;
    const int heads = min(G, heads_all - g0), head0 = h * heads_all + g0;
    const int b = request_of(p.query_start, p.batch, t, lane);
    if (b >= p.batch) return;
    const int kv_len = p.kv_lens[b], end = p.query_start ? p.query_start[b + 1] : t + 1;
    const Visible vis = paged::visible(kv_len - end + t, kv_len, p.held, p.window, p.sinks);
    const int keys = paged::run_of_keys(vis.count, p.shortest_run, p.max_runs), runs = max(1, (vis.count + keys - 1) / keys);
    if (run >= runs) return;
    const int lo = run * keys, hi = min(vis.count, lo + keys);

    float q[G][EL];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float *row = p.q + (size_t)t * p.q_row + (size_t)(head0 + min(g, heads - 1)) * p.q_head + EL * sub;
#pragma unroll
        for (int e = 0; e < EL; e += 4) {
            const float4 x = load4(row + e);
            q[g][e] = x.x * kQueryScale; q[g][e + 1] = x.y * kQueryScale; q[g][e + 2] = x.z * kQueryScale; q[g][e + 3] = x.w * kQueryScale;
        }
    }
    const int *table = p.tables + (size_t)b * p.width;
    constexpr int kBytes = 16 / EL;  // of an element
    const char *kb = static_cast<const char *>(p.k) + 16 * sub, *vb = static_cast<const char *>(p.v) + 16 * sub;
    float m[G], l[G], o[G][EL];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < EL; ++e) o[g][e] = 0.0f;
    }
    int id[PASS], off[PASS];
    auto pages = [&](int first) {
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            const int v = first + i * (W * KEYS), j = v < hi ? vis.key(v) : 0, at = p.div.page(j);
            off[i] = j - at * p.div.size;
            id[i] = v < hi ? table[at] : -1;
        }
    };
    const int first = lo + wave * KEYS + own;
    pages(first);
    for (int base = first - own; base < hi; base += PASS * W * KEYS) {
        uint4 kx[PASS], vx[PASS];
        bool ok[PASS];
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            ok[i] = (unsigned)id[i] < (unsigned)p.n_pages;
            const size_t row = (size_t)(h * p.div.size + (ok[i] ? off[i] : 0)) * DH, page = ok[i] ? id[i] : 0;
            kx[i] = *reinterpret_cast<const uint4 *>(kb + (page * p.k_page + row) * kBytes);
            vx[i] = *reinterpret_cast<const uint4 *>(vb + (page * p.v_page + row) * kBytes);
        }
        pages(base + own + PASS * W * KEYS);
        float s[G][PASS];
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            float f[EL];
            T::floats(kx[i], f);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float d = q[g][0] * f[0];
#pragma unroll
                for (int e = 1; e < EL; ++e) d = fmaf(q[g][e], f[e], d);
                s[g][i] = ok[i] ? sum_of_key<LPK>(d) : -INFINITY;
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float top = m[g];
#pragma unroll
            for (int i = 0; i < PASS; ++i) top = fmaxf(top, s[g][i]);
            const float ref = top == -INFINITY ? 0.0f : top, a = __builtin_amdgcn_exp2f(m[g] - ref);
            l[g] *= a;
#pragma unroll
            for (int e = 0; e < EL; ++e) o[g][e] *= a;
#pragma unroll
            for (int i = 0; i < PASS; ++i) {
                s[g][i] = __builtin_amdgcn_exp2f(s[g][i] - ref);
                l[g] += s[g][i];
            }
            m[g] = top;
        }
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            float f[EL];
            T::floats(vx[i], f);
#pragma unroll
            for (int e = 0; e < EL; ++e) {
                const float x = ok[i] ? f[e] : 0.0f;  // (what lies behind the keys may be no number)
#pragma unroll
                for (int g = 0; g < G; ++g) o[g][e] = fmaf(s[g][i], x, o[g][e]);
            }
        }
    }
    // the wave's keys together, then the waves
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float top = over_keys<LPK>(m[g], [](float a, float c) { return fmaxf(a, c); });
        const float f = m[g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[g] - top);
        const float sum = over_keys<LPK>(l[g] * f, [](float a, float c) { return a + c; });
#pragma unroll
        for (int e = 0; e < EL; ++e) {
            const float x = over_keys<LPK>(o[g][e] * f, [](float a, float c) { return a + c; });
            if (own == 0) s_o[wave][g][EL * sub + e] = x;
        }
        if (lane == 0) {
            s_m[wave][g] = top;
            s_l[wave][g] = sum;
        }
    }
    __syncthreads();
    auto place = [&](int r, int g) { return p.partial + (((size_t)item * p.max_runs + r) * G + g) * (DH + 2); };
    float *out = p.o + ((size_t)t * p.n_heads + head0) * DH + lane;
    for (int g = wave; g < heads; g += W) {
        float top = -INFINITY, acc = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w][g]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = s_m[w][g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[w][g] - top);
            acc = fmaf(s_o[w][g][lane], f, acc);
            sum = fmaf(s_l[w][g], f, sum);
        }
        if (runs == 1) {
            out[g * DH] = sum == 0.0f ? 0.0f : acc / sum;
        } else {
            float *part = place(run, g);
            __hip_atomic_store(part + lane, acc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (lane == 0) {
                __hip_atomic_store(part + DH, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(part + DH + 1, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
    if (runs == 1) return;
    __shared__ unsigned int s_ticket;
    partials_published(p.strict);
    __syncthreads();
    if (tid == 0) {
        s_ticket = take_ticket(&p.counters[item], p.strict);
        if (s_ticket == (unsigned)(runs - 1)) __hip_atomic_store(&p.counters[item], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s_ticket != (unsigned)(runs - 1)) return;
    if (p.strict) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    for (int g = wave; g < heads; g += W) {
        auto load = [&](int r, int i) { return __hip_atomic_load(place(r, g) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        // lane r: the weight of run r (and of r + 64, ...)
        float top = -INFINITY;
        for (int r = lane; r < runs; r += 64) top = fmaxf(top, load(r, DH));
        top = wave_max(top);
        float sum = 0.0f, acc = 0.0f;
        for (int r0 = 0; r0 < runs; r0 += 64) {
            const float mr = r0 + lane < runs ? load(r0 + lane, DH) : -INFINITY, f = mr == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mr - top);
            sum += wave_sum(r0 + lane < runs ? load(r0 + lane, DH + 1) * f : 0.0f);
            const int n = min(64, runs - r0);
            for (int r = 0; r < n; ++r) acc = fmaf(load(r0 + r, lane), __shfl(f, r, kWave), acc);
        }
        out[g * DH] = sum == 0.0f ? 0.0f : acc / sum;
    }
}

template <class T, int G>
int32_t tokens_go(agpu_ctx *ctx, PagedAttn &p, int64_t longest) {
    const int64_t items = (int64_t)p.tokens * p.n_kv * ceil_div(p.n_heads / p.n_kv, G);
    const paged::Cut cut = paged::cut_keys(items, longest, 2048, 128, 64, G * (DH + 2) * sizeof(float), ctx->ws_bytes / 2, ctx->n_counters - 1);
    p.shortest_run = cut.shortest;
    p.max_runs = cut.runs;
    hipLaunchKernelGGL((paged_tokens_kernel<T, G, 4, 4>), dim3((unsigned)items, cut.runs), dim3(256), 0, ctx->stream, p);
    return AGPU_LAUNCH_CHECK(ctx, "paged_tokens_kernel");
}
template <class T>
int32_t attention_go(agpu_ctx *ctx, PagedAttn &p, int64_t longest) {
    const int g = p.n_heads / p.n_kv;
    return g == 1 ? tokens_go<T, 1>(ctx, p, longest) : g == 2 ? tokens_go<T, 2>(ctx, p, longest) : g <= 4 ? tokens_go<T, 4>(ctx, p, longest) : tokens_go<T, 8>(ctx, p, longest);
}

}  // namespace

AGPU_EXPORT int32_t agpu_paged_attention(agpu_ctx *ctx, const float *q, int64_t q_token_stride, int64_t q_head_stride, const void *k_cache,
                                         const void *v_cache, int64_t k_page_stride, int64_t v_page_stride, const int32_t *block_tables,
                                         const int32_t *kv_lens, const int32_t *query_start, float *o, int32_t tokens, int32_t batch,
                                         int32_t n_heads, int32_t n_kv_heads, int32_t n_pages, int32_t page_size, int32_t table_width,
                                         int32_t window, int32_t sinks, int32_t d_head, int32_t cache_type) {
    AGPU_REQUIRE_CTX(ctx);
    const paged::Refusal cache =
        paged::refuse_cache((uintptr_t)k_cache, (uintptr_t)v_cache, k_page_stride, v_page_stride, n_kv_heads, n_pages, page_size, d_head, cache_type);
    paged::Refusal no = paged::refuse_attention(tokens, batch, n_heads, n_kv_heads, table_width, page_size, window, sinks, query_start != nullptr);
    if (no.code == AGPU_OK) no = cache;
    if (no.code != AGPU_OK) return agpu_fail(ctx, no.code, "paged_attention: %s", no.why);
    if (tokens == 0 || batch == 0) return AGPU_OK;
    if (!q || !k_cache || !v_cache || !kv_lens || !o || (!block_tables && table_width > 0))
        return agpu_fail(ctx, AGPU_ERR_NULL_POINTER, "paged_attention: null pointer");
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    PagedAttn p{};
    p.q = q; p.q_row = q_token_stride; p.q_head = q_head_stride;
    p.k = k_cache; p.v = v_cache; p.k_page = k_page_stride; p.v_page = v_page_stride;
    p.tables = block_tables; p.kv_lens = kv_lens; p.query_start = query_start; p.o = o;
    p.tokens = tokens; p.batch = batch; p.n_heads = n_heads; p.n_kv = n_kv_heads; p.n_pages = n_pages;
    p.width = table_width; p.held = table_width * page_size; p.window = window; p.sinks = sinks;
    p.div = PageDiv::of(page_size);
    p.partial = reinterpret_cast<float *>(ctx->workspace);
    p.counters = ctx->counters;
    p.strict = ctx->strict_sync;
    const int64_t longest = paged::longest_row(p.held, window, sinks);
    return cache_type == AGPU_CACHE_F32 ? attention_go<F32>(ctx, p, longest) : cache_type == AGPU_CACHE_F16 ? attention_go<F16>(ctx, p, longest) : attention_go<BF16>(ctx, p, longest);
}
