// The kernels of attention over a KV cache in pages (paged_attention.hip says what bounds them and how they are cut up), with what the operators beside it need of
// them besides: WEIGHTS (paged_weights.hip) keeps the rows' statistics and adds up how much weight each key was given; SHARED (paged_shared.hip) joins in what
// rows have seen of a prefix, and PREFIX is that part of the work.
#pragma once
#include "agpu_internal.h"
#include "gemm_bf16.h"
#include "paged.h"

#include <algorithm>
#include <type_traits>

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
    PageDiv div, group;  // by the page size, and by the heads of a K/V head
    int strict;
};

enum Mode { PLAIN, WEIGHTS, SHARED, PREFIX };

// What a kernel gets for what it does besides.
template <int MODE>
struct More {};
template <>
struct More<WEIGHTS> {
    float *weights;   // [n_pages][n_kv][page_size]
    long long page;   // elements between pages
    float *scores;    // of requests with one row: [batch][n_kv][seen][group], or, with seen = 0, [n_pages][n_kv][page_size][group]; null: there is no room for them
    int seen;         // the most keys that a row sees
    float2 *stats;    // [tokens][n_heads]: the unit of a row's weights and what they are divided by
    int at_once;      // tiles of a head's keys that are numbered at a time
    bool few;         // weights are added up from scores by the last workgroup at a token; otherwise, and without scores, by paged_weights_kernel
    __device__ __forceinline__ bool scored(int rows, int group) const { return rows == 1 && group <= 8 && scores != nullptr; }
    // Where the first score of request b's key number v is, which is at position `off` of a page (there are less than 2^32 scores).
    __device__ __forceinline__ uint32_t score_at(const PagedAttn &p, int b, int h, int v, int page, int off) const {
        const uint32_t size = seen ? seen : p.div.size;
        return ((uint32_t)((seen ? b : page) * p.n_kv + h) * size + (uint32_t)(seen ? v : off)) * (uint32_t)p.group.size;
    }
};
template <>
struct More<SHARED> {
    const int *tables, *lens, *of;  // of the prefixes [n_prefix][width], [n_prefix]; of the requests
    int n_prefix, width, held;
    // What rows have seen of their prefix, in runs: o of the first run is in first [tokens][n_heads][64], which is where the rows' results go if that begins at 16 bytes, of
    // the others in rest [runs - 1][tokens][n_heads][64]; (m, l) of all in ml [runs][tokens][n_heads].
    float *first, *rest;
    float2 *ml;
    int *before;  // [batch] how many runs there are of what a request's rows have seen of their prefix
    __device__ __forceinline__ int len(int g) const { return (unsigned)g < (unsigned)n_prefix ? max(min(lens[g], held), 0) : 0; }
};
template <>
struct More<PREFIX> : More<SHARED> {};

// How keys are cut into runs over workgroups, and where items of several runs leave their partial results and draw their tickets.
struct Runs {
    int run, most;  // about how many keys; how many runs at most
    float *partial;
    int part;  // floats of an item's run there
    unsigned int *counters;
};

// Scores are in units of the binary logarithm: q is taken times log2(e) / 8.
constexpr float kQueryScale = 0.125f * 1.44269504088896340736f;

// ---- elements of the cache, 16 bytes a lane ----
struct F32 {
    static constexpr int EL = 4;
    static __device__ __forceinline__ float one(const void *p, size_t i) { return static_cast<const float *>(p)[i]; }
    static __device__ __forceinline__ void floats(const uint4 &x, float (&f)[4]) {
        f[0] = __uint_as_float(x.x); f[1] = __uint_as_float(x.y); f[2] = __uint_as_float(x.z); f[3] = __uint_as_float(x.w);
    }
};
struct BF16 {
    static constexpr int EL = 8;
    static constexpr uint32_t kExponent = 0x7f80, kOdd = 217 << 7;  // the exponents' bits; those from which on an element is odd: 2^90
    static __device__ __forceinline__ float one(const void *p, size_t i) { return __uint_as_float((uint32_t)static_cast<const unsigned short *>(p)[i] << 16); }
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
    static constexpr uint32_t kExponent = 0x7c00, kOdd = 0x7c00;
    static __device__ __forceinline__ float one(const void *p, size_t i) { return (float)static_cast<const _Float16 *>(p)[i]; }
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

// The request that token t belongs to (uniform; `batch`: behind the last one, or before the first).
__device__ __forceinline__ int request_of(const int *query_start, int batch, int t, int lane) {
    if (!query_start) return t;
    if (t < batch && query_start[t] == t && query_start[t + 1] == t + 1) return t;  // one token each so far, as a rule
    int b = 0;
    for (int i = 0; i < batch; i += 64) b += __popcll(__ballot(i + lane < batch && query_start[i + lane + 1] <= t));
    return t < query_start[0] ? batch : b;
}

// The first positions that stay visible, of those on a request's own pages.
template <int MODE>
__device__ __forceinline__ int sinks_of(const PagedAttn &p, const More<MODE> &more, int b) {
    if constexpr (MODE == SHARED) return p.sinks > 0 ? max(p.sinks - more.len(more.of[b]), 0) : 0;
    return p.sinks;
}

// What a workgroup of W waves needs in LDS for a token's G query heads.
template <int G, int W>
struct TokenShared {
    float o[W][G][DH], m[W][G], l[W][G];
    unsigned int ticket;
};

// Up to G query heads of a token that share a K/V head over a run of its keys, by 64 W threads.  LPK lanes share a key, 16 bytes each.
// pos: the token's position in request b; h: K/V head, head0: first of the query heads, heads: how many; item: place among the partial results.
template <class T, int G, int W, int PASS, int MODE>
__device__ __forceinline__ void token_run(const PagedAttn &p, const More<MODE> &more, TokenShared<G, W> &s, const Runs &cut, int t, int b, int pos, int h, int head0, int heads, int run, int item) {
    constexpr int EL = T::EL, LPK = DH / EL, KEYS = 64 / LPK;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sub = lane % LPK, own = lane / LPK;
    const Visible vis = paged::visible(pos, pos + 1, p.held, p.window, sinks_of(p, more, b));
    const paged::RunsOf cuts = paged::runs_of(vis.count, cut.run, cut.most);
    const int runs = cuts.runs;
    if (run >= runs) return;
    const int lo = run * cuts.keys, hi = min(vis.count, lo + cuts.keys);

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
    bool scored = false, at_once = false;
    if constexpr (MODE == WEIGHTS) {
        scored = more.scored(p.query_start ? p.query_start[b + 1] - p.query_start[b] : 1, p.group.size);
        at_once = scored && more.few;
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
    // Scores leave when the next keys are on their way: loads wait for stores before them (64 requests of 4096 keys, 32 heads over 8, f16: 141 us, 126 this way, 110 without scores).
    float late[PASS];
    uint32_t late_to[PASS];
    auto store_late = [&] {
        if constexpr (MODE == WEIGHTS)
#pragma unroll
            for (int i = 0; i < PASS; ++i)
                if (late_to[i] != 0xffffffffu) __hip_atomic_store(more.scores + late_to[i], late[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    };
#pragma unroll
    for (int i = 0; i < PASS; ++i) late_to[i] = 0xffffffffu;
    const int first = lo + wave * KEYS + own;
    pages(first);
    for (int base = first - own; base < hi; base += PASS * W * KEYS) {
        uint4 kx[PASS], vx[PASS];
        bool ok[PASS];
        uint32_t key[PASS];  // where this lane's score goes
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            ok[i] = (unsigned)id[i] < (unsigned)p.n_pages;
            const size_t row = (size_t)(h * p.div.size + (ok[i] ? off[i] : 0)) * DH, page = ok[i] ? id[i] : 0;
            kx[i] = *reinterpret_cast<const uint4 *>(kb + (page * p.k_page + row) * kBytes);
            vx[i] = *reinterpret_cast<const uint4 *>(vb + (page * p.v_page + row) * kBytes);
            if constexpr (MODE == WEIGHTS) key[i] = scored && ok[i] && sub < heads ? more.score_at(p, b, h, base + own + i * (W * KEYS), id[i], off[i]) + sub : 0xffffffffu;
        }
        pages(base + own + PASS * W * KEYS);
        if constexpr (MODE == WEIGHTS) store_late();
        float x[G][PASS];
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            float f[EL];
            T::floats(kx[i], f);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float d = q[g][0] * f[0];
#pragma unroll
                for (int e = 1; e < EL; ++e) d = fmaf(q[g][e], f[e], d);
                x[g][i] = ok[i] ? sum_of_key<LPK>(d) : -INFINITY;
            }
            if constexpr (MODE == WEIGHTS) {  // (lanes of a key have its scores all, and there are at least as many as heads)
                late[i] = x[0][i];
#pragma unroll
                for (int g = 1; g < G; ++g) late[i] = sub == g ? x[g][i] : late[i];
                late_to[i] = key[i];
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float top = m[g];
#pragma unroll
            for (int i = 0; i < PASS; ++i) top = fmaxf(top, x[g][i]);
            const float ref = top == -INFINITY ? 0.0f : top, a = __builtin_amdgcn_exp2f(m[g] - ref);
            l[g] *= a;
#pragma unroll
            for (int e = 0; e < EL; ++e) o[g][e] *= a;
#pragma unroll
            for (int i = 0; i < PASS; ++i) {
                x[g][i] = __builtin_amdgcn_exp2f(x[g][i] - ref);
                l[g] += x[g][i];
            }
            m[g] = top;
        }
#pragma unroll
        for (int i = 0; i < PASS; ++i) {
            float f[EL];
            T::floats(vx[i], f);
#pragma unroll
            for (int e = 0; e < EL; ++e) {
                const float y = ok[i] ? f[e] : 0.0f;  // (what lies behind the keys may be no number)
#pragma unroll
                for (int g = 0; g < G; ++g) o[g][e] = fmaf(x[g][i], y, o[g][e]);
            }
        }
    }
    if constexpr (MODE == WEIGHTS) store_late();
    // What the rows have seen of a prefix counts as keys of the first run: lanes of a key take a run of it each, as many as there are.  (Loaded before the keys it would cost a wave
    // of five on a SIMD: 64 requests, 25 heads 18.6 us, 16.9.)
    if constexpr (MODE == SHARED) {
        const int before = run == 0 ? more.before[b] : 0;
        const size_t rows = (size_t)p.tokens * p.n_heads;
        for (int r = wave + W * own; r < before; r += W * KEYS)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const size_t row = (size_t)t * p.n_heads + head0 + min(g, heads - 1);
                const float *from = (r == 0 ? more.first + row * DH : more.rest + ((r - 1) * rows + row) * DH) + EL * sub;
                const float2 ml = more.ml[r * rows + row];
                const float now = fmaxf(m[g], ml.x), keep = m[g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[g] - now), f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - now);
                m[g] = now;
                l[g] = fmaf(ml.y, f, l[g] * keep);
#pragma unroll
                for (int e = 0; e < EL; e += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(from + e);
                    o[g][e] = fmaf(x.x, f, o[g][e] * keep); o[g][e + 1] = fmaf(x.y, f, o[g][e + 1] * keep);
                    o[g][e + 2] = fmaf(x.z, f, o[g][e + 2] * keep); o[g][e + 3] = fmaf(x.w, f, o[g][e + 3] * keep);
                }
            }
    }
    // The wave's keys together: the rows of 16 lanes are added in two steps that halve the values a lane has, so that each row ends with a quarter of them;
    // then the waves.
    constexpr int N = G * EL;
    float y[N];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float top = over_keys<LPK>(m[g], [](float a, float c) { return fmaxf(a, c); });
        const float f = m[g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[g] - top);
        const float sum = over_keys<LPK>(l[g] * f, [](float a, float c) { return a + c; });
        if (lane == 0) {
            s.m[wave][g] = top;
            s.l[wave][g] = sum;
        }
#pragma unroll
        for (int e = 0; e < EL; ++e) y[g * EL + e] = o[g][e] * f;
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(y[i]), __float_as_uint(y[i + N / 2]), false, false);
        y[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(y[i]), __float_as_uint(y[i + N / 4]), false, false);
        y[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        if (LPK == 8) y[i] += dpp_move<0x128, 0xf>(0.0f, y[i]);  // row_ror:8
        const int n = i + N / 4 * (lane >> 4 & 1) + N / 2 * (lane >> 5);
        if (LPK == 16 || (lane & 8) == 0) s.o[wave][n / EL][EL * sub + n % EL] = y[i];
    }
    __syncthreads();
    auto place = [&](int r, int g) { return cut.partial + ((size_t)item * cut.most + r) * cut.part + g * (DH + 2); };
    float *out = p.o + ((size_t)t * p.n_heads + head0) * DH + lane;
    // A head's result, and what there is to do besides.
    auto finish = [&](int g, float acc, float top, float sum) {
        out[g * DH] = sum == 0.0f ? 0.0f : acc / sum;
        if constexpr (MODE == WEIGHTS) {
            const float unit = top == -INFINITY ? 0.0f : top, share = sum == 0.0f ? 0.0f : 1.0f / sum;
            if (lane != 0) return;
            if (at_once) s.m[0][g] = unit, s.l[0][g] = share;  // (this wave alone has read what was there)
            else more.stats[(size_t)t * p.n_heads + head0 + g] = make_float2(unit, share);
        }
    };
    // The only row of its request: what each key was given, from the scores that all workgroups at it have left.
    auto add_weights = [&] {
        if constexpr (MODE == WEIGHTS) {
            if (!at_once) return;
            __syncthreads();
            constexpr int KEYS_AT_ONCE = 4;  // what is loaded is loaded together
            for (int v0 = tid; v0 < vis.count; v0 += KEYS_AT_ONCE * 64 * W) {
                int place[KEYS_AT_ONCE], page[KEYS_AT_ONCE];
                float x[KEYS_AT_ONCE][G], old[KEYS_AT_ONCE];
#pragma unroll
                for (int k = 0; k < KEYS_AT_ONCE; ++k) {
                    const int v = v0 + k * 64 * W, j = v < vis.count ? vis.key(v) : 0, at = p.div.page(j);
                    place[k] = h * p.div.size + (j - at * p.div.size);
                    page[k] = v < vis.count ? table[at] : -1;
                }
#pragma unroll
                for (int k = 0; k < KEYS_AT_ONCE; ++k) {
                    const bool there = (unsigned)page[k] < (unsigned)p.n_pages;
                    page[k] = there ? page[k] : -1;
                    const size_t of = there ? page[k] : 0;
                    const float *const score = more.scores + more.score_at(p, b, h, min(v0 + k * 64 * W, vis.count - 1), (int)of, place[k] - h * p.div.size);
#pragma unroll
                    for (int g = 0; g < G; ++g) x[k][g] = __hip_atomic_load(score + min(g, heads - 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    old[k] = more.weights[of * more.page + place[k]];
                }
#pragma unroll
                for (int k = 0; k < KEYS_AT_ONCE; ++k) {
                    if (page[k] < 0) continue;
                    float sum = 0.0f;
#pragma unroll
                    for (int g = 0; g < G; ++g) sum += g < heads ? __builtin_amdgcn_exp2f(x[k][g] - s.m[0][g]) * s.l[0][g] : 0.0f;
                    const int v = v0 + k * 64 * W;
                    more.weights[page[k] * more.page + place[k]] = (vis.key(v) == pos ? 0.0f : old[k]) + sum;
                }
            }
        }
    };
    for (int g = wave; g < heads; g += W) {
        float top = -INFINITY, acc = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, s.m[w][g]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = s.m[w][g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s.m[w][g] - top);
            acc = fmaf(s.o[w][g][lane], f, acc);
            sum = fmaf(s.l[w][g], f, sum);
        }
        if (runs == 1) {
            finish(g, acc, top, sum);
        } else {
            float *part = place(run, g);
            __hip_atomic_store(part + lane, acc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (lane == 0) {
                __hip_atomic_store(part + DH, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(part + DH + 1, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
    if (runs == 1) {
        if constexpr (MODE == WEIGHTS) partials_published(p.strict);  // (the scores, for the workgroup's other waves)
        return add_weights();
    }
    partials_published(p.strict);
    __syncthreads();
    if (tid == 0) {
        s.ticket = take_ticket(&cut.counters[item], p.strict);
        if (s.ticket == (unsigned)(runs - 1)) __hip_atomic_store(&cut.counters[item], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s.ticket != (unsigned)(runs - 1)) return;
    if (p.strict) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    for (int g = wave; g < heads; g += W) {
        auto load = [&](int r, int i) { return __hip_atomic_load(place(r, g) + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        // lane r: the weight of run r (there are 64 at most).  All that is wanted first goes on its way together, eight runs' sums among it, which the compiler would take
        // one by one.
        const float mr = lane < runs ? load(lane, DH) : -INFINITY, lr = lane < runs ? load(lane, DH + 1) : 0.0f;
        float x[8];
        auto eight = [&](int r) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = load(min(r + e, runs - 1), lane);
            __builtin_amdgcn_sched_barrier(0);
        };
        eight(0);
        const float top = wave_max(mr), f = mr == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mr - top), sum = wave_sum(lr * f);
        float acc = 0.0f;
        for (int r = 0; r < runs; r += 8) {
            if (r > 0) eight(r);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc = r + e < runs ? fmaf(x[e], __shfl(f, r + e, kWave), acc) : acc;
        }
        finish(g, acc, top, sum);
    }
    add_weights();
}

constexpr int kListed = 256;
// The work of up to 256 entries (requests, or tokens), in LDS: running sums of their units.  A workgroup numbers all units, entry by entry, and takes
// those of its own number, that plus the number of workgroups, and so on.
struct Units {
    int incl[kListed];
    // units[j] of entry 64 j + lane, the same in every wave; returns how many there are (a barrier has to follow)
    __device__ __forceinline__ int number(const int (&units)[4], int entries, int lane) {
        int all = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (64 * j >= entries) break;  // uniform
            const int v = wave_running_sum(units[j]);
            incl[64 * j + lane] = v + all;
            all += __builtin_amdgcn_readlane(v, 63);
        }
        return all;
    }
    // the entry of unit u; u becomes its number within the entry
    __device__ __forceinline__ int entry(int &u, int lane) const {
        int at = 0, before = 0;
        for (int j = 0;; ++j) {
            const int v = incl[64 * j + lane];
            const uint64_t beyond = __ballot(v > u);
            if (beyond != 0) {  // uniform; there is one
                at = __builtin_ctzll(beyond);
                if (at > 0) before = __builtin_amdgcn_readlane(v, at - 1);
                u -= before;
                return 64 * j + at;
            }
            before = __builtin_amdgcn_readlane(v, 63);
        }
    }
};

// What the last row of a request (or a tile of `rows` tokens) sees at most.
__device__ __forceinline__ int keys_seen(const PagedAttn &p, int kv_len, int rows) {
    const int held = max(min(kv_len, p.held), 0);
    return p.window > 0 ? (int)min((long long)held, (long long)p.window + p.sinks + rows) : held;
}

// Two runs' worth of keys a CU (fewer, longer runs are joined less often: 64 tokens of 4096 keys 124 us with four, 104 with two).
// Every row by itself, whatever request it belongs to: a unit is a run of the keys of up to G query heads of a token that share a K/V head.  Up to 256 tokens
// (`listed`) the units are numbered and a run is as long as it takes to keep the device busy; for more, there are items * cut.most.
template <class T, int G, int W, int PASS, int MODE>
__global__ __launch_bounds__(64 * W) void paged_tokens_kernel(const PagedAttn p, Runs cut, float fill, int least, int listed, const More<MODE> more) {
    __shared__ TokenShared<G, W> s;
    __shared__ Units list;
    __shared__ int owners[kListed], positions[kListed];
    const int lane = threadIdx.x & 63, heads_all = p.n_heads / p.n_kv, blocks = (heads_all + G - 1) / G;  // (G is the power of two that covers them, up to 8)
    const int per_token = p.n_kv * blocks;
    int all = p.tokens * per_token * cut.most;
    if (listed) {
        int units[4], longest = 0;
        float work = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            units[j] = 0;
            if (64 * j >= p.tokens) continue;  // uniform
            const int row = 64 * j + lane;
            if (row < p.tokens) {
                // the request of a row that is no request's only one: its first entry of query_start beyond the row
                int b = row;
                if (p.query_start && !(row < p.batch && p.query_start[row] == row && p.query_start[row + 1] == row + 1)) {
                    int lo = 0, hi = p.batch;
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (p.query_start[mid + 1] <= row) lo = mid + 1;
                        else hi = mid;
                    }
                    b = row < p.query_start[0] ? p.batch : lo;
                }
                if (b < p.batch) {
                    const int kv_len = max(p.kv_lens[b], 0);
                    owners[row] = b;
                    positions[row] = kv_len - (p.query_start ? p.query_start[b + 1] : row + 1) + row;
                    units[j] = max(keys_seen(p, kv_len, 1), 1);
                }
            }
            work += (float)units[j];
            longest = max(longest, units[j]);
        }
        cut.run = paged::run_for(wave_sum(work) * per_token, fill, least, (int)wave_minmax_u32<true>((unsigned)longest), cut.most);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (64 * j < p.tokens) units[j] = units[j] > 0 ? paged::runs_of(units[j], cut.run, cut.most).runs * per_token : 0;
        all = list.number(units, p.tokens, lane);
    }
    for (int unit = blockIdx.x; unit < all; unit += gridDim.x) {
        __syncthreads();  // the numbers, and what the last unit left
        int at = unit, t, run, hb, b, pos;
        if (listed) {
            t = list.entry(at, lane);
            run = at / per_token;
            hb = at - run * per_token;
            b = owners[t];
            pos = positions[t];
        } else {
            run = at % cut.most;
            at /= cut.most;
            t = at / per_token;
            hb = at - t * per_token;
            b = request_of(p.query_start, p.batch, t, lane);
            if (b >= p.batch) continue;
            pos = max(p.kv_lens[b], 0) - (p.query_start ? p.query_start[b + 1] : t + 1) + t;
        }
        const int h = hb / blocks, g0 = (hb - h * blocks) * G;
        token_run<T, G, W, PASS>(p, more, s, cut, t, b, pos, h, h * heads_all + g0, min(G, heads_all - g0), run, t * per_token + hb);
    }
}

// ---- tiles of rows on the matrix cores ----
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16 with 32 keys and 32 rows: what a 32 x 32 result holds of a column (a row of q) in its two
// half waves is what the second product takes, if V's keys come in the order 16 step + 8 (e / 4) + 4 half + e mod 4.
//   fp32 cache   every operand is the exact sum of three bf16 numbers (8 bits each, cut off one after the other); of the nine products of pieces the three
//                smallest are left out, which come to 2^-21 of the whole at most (2^-24.5 on average, always of its sign); the others, the smallest first.  All nine
//                would be half as many matrix instructions again for less than what the sums' own roundings are.
//   bf16 cache   K and V as they are, q and the weights in three pieces: three products, nothing left out
//   f16 cache    K and V as they are, q (times a power of two per row) and the weights (times 2^9) as two f16 numbers: two products.  q is good to 2^-22 of itself
//                and 2^-39 of its row's largest element, a weight to 2^-22 of itself and 2^-34 of the largest one (f16 has no steps below 2^-24): keys of weights below
//                that reach the sum of weights, which is fp32, but not o.  A third piece would be half as many products again.
constexpr int TILE_ROWS = 128, TILE_KEYS = 32;
constexpr int kFrag = 4 * 2 * 32;  // 16-byte fragments of a piece of 32 keys of K, and of V
typedef float floatx16 __attribute__((ext_vector_type(16)));

// Where in LDS the 16 elements `part` of the row of V of a key lie, in bytes: 128 a key, its four parts in an order by which eight keys' parts, which are
// read at a time, come from different banks.
__device__ __forceinline__ int tile_v_at(int key, int part) { return 128 * key + 32 * (part ^ (key & 2) ^ (key >> 2 & 1)); }

__device__ __forceinline__ uint32_t upper_halves(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }
__device__ __forceinline__ float without_top(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// Eight floats -> their three pieces, the largest first
__device__ __forceinline__ void pieces_of(const float (&v)[8], uint4 (&piece)[3]) {
    float r[8], t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        r[e] = without_top(v[e]);
        t[e] = without_top(r[e]);
    }
    piece[0] = make_uint4(upper_halves(v[0], v[1]), upper_halves(v[2], v[3]), upper_halves(v[4], v[5]), upper_halves(v[6], v[7]));
    piece[1] = make_uint4(upper_halves(r[0], r[1]), upper_halves(r[2], r[3]), upper_halves(r[4], r[5]), upper_halves(r[6], r[7]));
    piece[2] = make_uint4(upper_halves(t[0], t[1]), upper_halves(t[2], t[3]), upper_halves(t[4], t[5]), upper_halves(t[6], t[7]));
}
__device__ __forceinline__ void pieces_of(const float (&v)[8], uint4 (&piece)[2]) {  // f16
    f16x8 hi, lo;
    split_f16(v, 1.0f, hi, lo);
    piece[0] = __builtin_bit_cast(uint4, hi);
    piece[1] = __builtin_bit_cast(uint4, lo);
}

template <class T>
struct Tiles;  // KP pieces of K and V, QP of q and the weights; UP: what weights are multiplied by
template <>
struct Tiles<F32> {
    static constexpr int KP = 3, QP = 3;
    static constexpr float UP = 1.0f;
    static __device__ __forceinline__ floatx16 mfma(uint4 a, uint4 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Tiles<BF16> {
    static constexpr int KP = 1, QP = 3;
    static constexpr float UP = 1.0f;
    static __device__ __forceinline__ floatx16 mfma(uint4 a, uint4 b, floatx16 c) { return Tiles<F32>::mfma(a, b, c); }
};
template <>
struct Tiles<F16> {
    static constexpr int KP = 1, QP = 2;
    static constexpr float UP = 512.0f;
    static __device__ __forceinline__ floatx16 mfma(uint4 a, uint4 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Eight elements of a key's row of K or V on their way from the cache to LDS.
template <class T>
struct Staged;
template <>
struct Staged<F32> {
    float x[8];
    __device__ __forceinline__ void row(const char *p) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 16);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    }
    __device__ __forceinline__ bool odd() const {  // one of them is infinite, no number, or larger than 2^91 (none of them, if all are below 2^87)
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) t = fmaf(x[e], 0x1p38f, t);
        return !(fabsf(t) < INFINITY);
    }
    // Zeros in place of what is infinite or no number; which they were.
    __device__ __forceinline__ uint32_t clean() {
        uint32_t odd = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (!(fabsf(x[e]) < INFINITY)) {
                odd |= 1u << e;
                x[e] = 0.0f;
            }
        return odd;
    }
    __device__ __forceinline__ void pieces(uint4 (&piece)[3]) const { pieces_of(x, piece); }
    __device__ __forceinline__ void store(uint4 *to) const {
        uint4 piece[3];
        pieces_of(x, piece);
#pragma unroll
        for (int i = 0; i < 3; ++i) to[i * kFrag] = piece[i];
    }
};
template <class T>
struct Staged16 {
    uint32_t x[4];  // two elements each
    __device__ __forceinline__ void row(const char *p) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    }
    __device__ __forceinline__ void clear() { x[0] = x[1] = x[2] = x[3] = 0; }
    __device__ __forceinline__ bool odd() const {  // with what is left up to the sign bit added, an exponent from kOdd on reaches it
        constexpr uint32_t ones = T::kExponent * 0x10001u, rest = (0x8000u - T::kOdd) * 0x10001u;
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) t |= (x[e] & ones) + rest;
        return (t & 0x80008000u) != 0;
    }
    __device__ __forceinline__ uint32_t clean() {
        uint32_t odd = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if ((x[e >> 1] >> (16 * (e & 1)) & T::kExponent) == T::kExponent) {
                odd |= 1u << e;
                x[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
            }
        return odd;
    }
    __device__ __forceinline__ void pieces(uint4 (&piece)[1]) const { piece[0] = make_uint4(x[0], x[1], x[2], x[3]); }
    __device__ __forceinline__ void store(uint4 *to) const { *to = make_uint4(x[0], x[1], x[2], x[3]); }
};
template <>
struct Staged<BF16> : Staged16<BF16> {};
template <>
struct Staged<F16> : Staged16<F16> {};

template <class T>
struct TileShared {
    uint4 k[2][Tiles<T>::KP][kFrag], v[2][Tiles<T>::KP][kFrag];  // [buffer][piece]: K [d step of 16][half][key], V [key][dimension], what tile_v_at says
    long long at[2][8][TILE_KEYS];  // of the keys of eight tiles: where their rows of K and of V begin, in bytes (0 for those that are not there)
    uint32_t seen[8];               // which of them are there
    uint32_t odd_k[8], odd_v[8];    // of which something is infinite or not a number, or of V so large that weights above one could take it beyond the largest number
    unsigned int ticket;
};

__device__ __forceinline__ float other_half(float v, float &own) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    own = __uint_as_float(r[0]);
    return __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_of_halves(float v) {
    float own;
    const float other = other_half(v, own);
    return fmaxf(own, other);
}
__device__ __forceinline__ float sum_of_halves(float v) {
    float own;
    const float other = other_half(v, own);
    return own + other;
}

// The rows of a tile's request: its tokens from `start` on are at positions from `first` on.
template <int MODE>
struct TileOf {
    int start, tokens, first;
    __device__ __forceinline__ int token(int i) const { return start + i; }
    __device__ __forceinline__ int pos(int i) const { return first + i; }
};
// The rows behind a prefix: tokens of any requests, those of this tile (from `first` on) listed in LDS.
template <>
struct TileOf<PREFIX> {
    const int *list, *positions;
    int first, tokens;
    __device__ __forceinline__ int token(int i) const { return list[i - first]; }
    __device__ __forceinline__ int pos(int i) const { return positions[i - first]; }
    int pos0, pos1;  // the smallest and the largest of the tile's positions
};

// Up to 128 rows of a request (its tokens' heads of one K/V head, token by token) over a run of the keys that any of them sees, by four waves of 32 rows, which
// share the tiles of 32 keys: what each thread has fetched goes to LDS as operands while the next tile is on its way, one barrier a tile (3200 cycles for a
// 16-bit cache, 4900 for an fp32 one).
// first_row: of the rows of the request (or of all behind a prefix) and K/V head; b: the request, or the prefix.
template <class T, int MODE>
__device__ __forceinline__ void tile_run(const PagedAttn &p, const More<MODE> &more, TileShared<T> &s, const Runs &cut, int b, const TileOf<MODE> &of, int h, int first_row, int run, int item) {
    constexpr int KP = Tiles<T>::KP, QP = Tiles<T>::QP;
    constexpr int kBytes = 16 / T::EL;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, h2 = lane >> 5;
    const int group = p.group.size, rows = of.tokens * group, last_row = min(first_row + TILE_ROWS, rows) - 1;
    // all keys that a row of the tile sees, numbered without a gap
    const int sinks = sinks_of(p, more, b);
    int held = p.held;
    if constexpr (MODE == PREFIX) held = more.len(b);
    int pos0, pos1;
    if constexpr (MODE == PREFIX) pos0 = of.pos0, pos1 = of.pos1;
    else pos0 = of.first + p.group.page(first_row), pos1 = of.first + p.group.page(last_row);
    const paged::TileKeys keys = paged::tile_keys(pos0, pos1, held, p.window, sinks);
    const int gap = keys.gap;
    const paged::RunsOf cuts = paged::runs_of(MODE == PREFIX ? held : keys.count, cut.run, cut.most);  // (of a prefix the same for all rows)
    const int runs = cuts.runs;
    if (run >= runs) return;
    const int lo = run * cuts.keys, hi = min(keys.count, lo + cuts.keys);
    // this lane's row; rows behind the last one repeat it
    const int row = min(first_row + 32 * wave + c, last_row), token = p.group.page(row), head = h * group + (row - token * group);
    const bool mine = first_row + 32 * wave + c <= last_row, any = first_row + 32 * wave <= last_row;
    const int t = of.token(token), pos = of.pos(token);
    int wave_pos0 = of.pos(p.group.page(min(first_row + 32 * wave, last_row))), wave_pos1 = of.pos(p.group.page(min(first_row + 32 * wave + 31, last_row)));
    if constexpr (MODE == PREFIX) wave_pos0 = pos0, wave_pos1 = pos1;  // (those of requests in no order)
    // which keys the row sees, and below which of those that are no sinks its wave's last row sees none
    const paged::RowKeys see = paged::row_keys(keys, pos, p.window, sinks);
    const int wave_low = paged::row_keys(keys, wave_pos1, p.window, sinks).low;

    // keys of tile i are lo + 32 i ..; their places are looked up for four tiles at a time, one a wave, long before they are fetched
    const int tiles = (hi - lo + TILE_KEYS - 1) / TILE_KEYS;
    const int *table = p.tables + (size_t)b * p.width;
    int id, off;
    auto look_up = [&](int i) {
        const int v = lo + TILE_KEYS * i + c;
        id = -1;
        off = 0;
        if (v < hi) {
            const int j = keys.key(v), page = p.div.page(j);
            id = table[page];
            off = j - page * p.div.size;
        }
    };
    auto leave = [&](int i) {  // a half wave for K, the other for V
        const bool ok = (unsigned)id < (unsigned)p.n_pages;
        s.at[h2][i & 7][c] = ok ? (id * (h2 ? p.v_page : p.k_page) + (long long)(h * p.div.size + off) * DH) * kBytes : 0;
        const uint64_t who = __ballot(ok);
        if (lane == 0) {
            s.seen[i & 7] = (uint32_t)who;
            s.odd_k[i & 7] = s.odd_v[i & 7] = 0;
        }
    };
    look_up(wave);

    const float *q_row = p.q + (size_t)t * p.q_row + (size_t)head * p.q_head;
    uint4 q[4][QP];
    float unit = 1.0f;  // of the scores
    {
        float x[4][8], most = 0.0f;
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) {
            const float4 a = load4(q_row + 16 * ds + 8 * h2), d = load4(q_row + 16 * ds + 8 * h2 + 4);
            const float y[8] = {a.x, a.y, a.z, a.w, d.x, d.y, d.z, d.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[ds][e] = y[e] * kQueryScale;
                most = fmaxf(most, fabsf(x[ds][e]));
            }
        }
        if (QP == 2) {  // into 2^14 .. 2^15
            const int up = max(min(141 - (int)((__float_as_uint(max_of_halves(most)) >> 23) & 255u), 100), -112);
            const float by = __uint_as_float((uint32_t)(up + 127) << 23);
            unit = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int ds = 0; ds < 4; ++ds)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[ds][e] *= by;
        }
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) pieces_of(x[ds], q[ds]);
    }

    leave(wave);
    look_up(4 + wave);
    __syncthreads();
    const char *const kb = static_cast<const char *>(p.k), *const vb = static_cast<const char *>(p.v);
    Staged<T> sk, sv;
    // What this thread fetches: eight elements of K and of V of key c.
    const int row_byte = (16 * wave + 8 * h2) * kBytes, v_at = tile_v_at(c, wave) + 16 * h2;
    auto fetch = [&](int i) {
        sk.row(kb + s.at[0][i & 7][c] + row_byte);
        sv.row(vb + s.at[1][i & 7][c] + row_byte);
    };
    // The operand of V: of dimension 32 db + c the keys tile_key(st, h2, 0..7), four rows at a time that ds_read_b64_tr_b16 turns (16 lanes read four rows of 16
    // elements, a row in four lanes, and each gets a column).
    const int turned = tile_v_at(4 * h2 + ((lane & 15) >> 2), c >> 4) + 8 * (lane & 3);
    auto v_operand = [&](const uint4 *piece, int st, int db) {
        typedef short four __attribute__((ext_vector_type(4)));
        const char *const at = reinterpret_cast<const char *>(piece) + (turned ^ (64 * db)) + 2048 * st;
        typedef __attribute__((address_space(3))) four *lds;
        const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)at)), d = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(at + 1024)));
        return make_uint4(a.x, a.y, d.x, d.y);
    };
    if (tiles > 0) fetch(0);

    floatx16 o[2] = {};
    float m = -INFINITY, l = 0.0f;
    for (int i = 0; i < tiles; ++i) {
        const int buf = i & 1;
        const uint32_t there = s.seen[i & 7];
        if (there != 0xffffffffu) {  // uniform; zeros instead of what is not there
            if (!(there >> c & 1)) {
                sk.clear();
                sv.clear();
            }
        }
        if (__builtin_expect(__any(sk.odd() || sv.odd()), 0)) {
            if (sk.clean()) atomicOr(&s.odd_k[i & 7], 1u << c);
            if (sv.odd()) atomicOr(&s.odd_v[i & 7], 1u << c);
            sv.clean();
        }
        sk.store(&s.k[buf][0][(2 * wave + h2) * 32 + c]);
        sv.store(&s.v[buf][0][v_at / 16]);
        if (i + 1 < tiles) fetch(i + 1);
        __syncthreads();
        if ((i & 3) == 0) {
            leave(i + 4 + wave);
            look_up(i + 8 + wave);
        }
        const int v0 = lo + TILE_KEYS * i;
        if (!any || (v0 >= keys.first && v0 > wave_pos1 - gap)) continue;  // (the next tile goes to the other buffer)
        floatx16 x = {};
#pragma unroll
        for (int level = QP - 1; level >= 0; --level)
#pragma unroll
            for (int ds = 0; ds < 4; ++ds)
#pragma unroll
                for (int kp = KP - 1; kp >= 0; --kp)
                    if (level - kp >= 0 && level - kp < QP) x = Tiles<T>::mfma(s.k[buf][kp][(2 * ds + h2) * 32 + c], q[ds][level - kp], x);
        if (QP == 2)
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] *= unit;
        // Keys with something infinite in them, or no number, went as zeros, which no row's other keys notice; their scores are formed in fp32 here, and
        // their values are added below, for the rows that see them.
        const uint32_t odd_k = s.odd_k[i & 7], odd_v = s.odd_v[i & 7];
        if (__builtin_expect(odd_k != 0, 0))
#pragma unroll 1
            for (int kk = 0; kk < TILE_KEYS; ++kk) {
                if (!(odd_k >> kk & 1)) continue;
                int h2 = lane >> 5;
                asm volatile("" : "+v"(h2));  // (what follows from it is worked out here, and takes no registers all along)
                const size_t at = (size_t)s.at[0][i & 7][kk];
                float d = 0.0f;
#pragma unroll 1
                for (int e = 0; e < 32; ++e) d = fmaf(q_row[32 * h2 + e] * kQueryScale, T::one(kb + at, 32 * h2 + e), d);
                d = sum_of_halves(d);
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = 8 * (r >> 2) + 4 * h2 + (r & 3) == kk ? d : x[r];
            }
        // only tiles at the ends of what rows see hide anything (uniform over the wave)
        const bool whole = there == 0xffffffffu && v0 + TILE_KEYS - 1 <= wave_pos0 - gap &&
                           (v0 > wave_low || v0 + TILE_KEYS <= see.first);
        auto in_sight = [&] {  // of this row, one bit a key
            auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; };  // bits 0 .. n - 1
            return there & below(see.last + 1 - v0) & (~below(see.low + 1 - v0) | below(see.first - v0));
        };
        if (!whole) {
            const uint32_t seen = in_sight() >> (4 * h2);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t all = (uint32_t)((int)(seen << (31 - 8 * (r >> 2) - (r & 3))) >> 31);
                x[r] = __uint_as_float((all & __float_as_uint(x[r])) | (~all & 0xff800000u));
            }
        }
        float top = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
        top = max_of_halves(top);
        // Weights may grow to 2^6 before everything is rescaled, but not beside values from 2^91 on: those go in with weights of one at most, as they do row by
        // row, so that their sums are finite where |v| times the keys is below 2^128.  (Sums of 2^30 smaller ones are finite anyway, and f16 values are small.)
        // Each row by what it sees itself: keys that only other rows of the tile see leave its bits as they are.
        float slack = 6.0f;
        if (__builtin_expect(!std::is_same_v<T, F16> && odd_v != 0, 0)) slack = (odd_v & in_sight()) != 0 ? 0.0f : slack;
        const bool rises = top > m + slack;
        if (__any(rises)) {
            const float now = rises ? top : m, a = now == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= a;
#pragma unroll
            for (int db = 0; db < 2; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] *= a;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[r] = __builtin_amdgcn_exp2f(x[r] - ref);
            sum += x[r];
        }
        l += sum;
        uint4 w[2][QP];
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[8 * st + e] * Tiles<T>::UP;
            pieces_of(y, w[st]);
        }
#pragma unroll
        for (int level = QP - 1; level >= 0; --level)
#pragma unroll
            for (int kp = KP - 1; kp >= 0; --kp)
                if (level - kp >= 0 && level - kp < QP)
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int db = 0; db < 2; ++db) o[db] = Tiles<T>::mfma(v_operand(s.v[buf][kp], st, db), w[st][level - kp], o[db]);
        if (__builtin_expect(odd_v != 0, 0))
#pragma unroll 1
            for (int kk = 0; kk < TILE_KEYS; ++kk) {
                const int v = v0 + kk;
                if (!(odd_v >> kk & 1)) continue;
                int h2 = lane >> 5;
                asm volatile("" : "+v"(h2));
                const bool sees = see.sees(v);
                float weight = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) weight = 8 * (r >> 2) + 4 * h2 + (r & 3) == kk ? x[r] : weight;
                weight = sum_of_halves(weight);  // (one of them is zero)
                const size_t at = (size_t)s.at[1][i & 7][kk];
#pragma unroll
                for (int db = 0; db < 2; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float y = T::one(vb + at, 32 * db + 8 * (r >> 2) + 4 * h2 + (r & 3));
                        o[db][r] += sees && !(fabsf(y) < INFINITY) ? weight * y : 0.0f;
                    }
            }
    }
    l = sum_of_halves(l);
    const size_t row_at = (size_t)t * p.n_heads + head;
    if constexpr (MODE == PREFIX) {
        if (!mine) return;
        const size_t rows_all = (size_t)p.tokens * p.n_heads;
        float *const out = (run == 0 ? more.first + row_at * DH : more.rest + ((run - 1) * rows_all + row_at) * DH) + 4 * h2;
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<float4 *>(out + 32 * db + 2 * r) = make_float4(o[db][r] / Tiles<T>::UP, o[db][r + 1] / Tiles<T>::UP, o[db][r + 2] / Tiles<T>::UP, o[db][r + 3] / Tiles<T>::UP);
        if (h2 == 0) more.ml[run * rows_all + row_at] = make_float2(m, l);
        return;
    }
    auto store = [&](float sum) {
        if (!mine) return;
        if constexpr (MODE == SHARED) {
            const int pre = more.before[b];
            const size_t rows_all = (size_t)p.tokens * p.n_heads;
            for (int i = 0; i < pre; ++i) {
                const float2 ml = more.ml[i * rows_all + row_at];
                const float *const from = (i == 0 ? more.first + row_at * DH : more.rest + ((i - 1) * rows_all + row_at) * DH) + 4 * h2;
                float4 x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = *reinterpret_cast<const float4 *>(from + 8 * e);
                const float now = fmaxf(m, ml.x), keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - now), f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - now);
                m = now;
                sum = fmaf(ml.y, f, sum * keep);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y[4] = {x[e].x, x[e].y, x[e].z, x[e].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[e >> 2][4 * (e & 3) + k] = fmaf(y[k], f * Tiles<T>::UP, o[e >> 2][4 * (e & 3) + k] * keep);
                }
            }
        }
        const float by = sum == 0.0f ? 0.0f : 1.0f / (sum * Tiles<T>::UP);
        if constexpr (MODE == WEIGHTS)
            if (h2 == 0) more.stats[row_at] = make_float2(m == -INFINITY ? 0.0f : m, sum == 0.0f ? 0.0f : 1.0f / sum);
        float *out = p.o + row_at * DH + 4 * h2;
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
#pragma unroll
                for (int e = 0; e < 4; ++e) out[32 * db + 2 * r + e] = sum == 0.0f ? 0.0f : o[db][r + e] * by;
    };
    if (runs == 1) return store(l);
    auto part = [&](int r) { return cut.partial + ((size_t)item * cut.most + r) * cut.part + wave * (32 * (DH + 2)); };  // [wave][two dimensions, or m and l][row]
    auto pair = [](float a, float b) { return (unsigned long long)__float_as_uint(b) << 32 | __float_as_uint(a); };
    auto place = [&](int r, int d) { return reinterpret_cast<unsigned long long *>(part(r)) + (d >> 1) * 32 + c; };  // of dimensions d and d + 1 of row c
    if (any) {
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int r = 0; r < 16; r += 2)
                __hip_atomic_store(place(run, 32 * db + 8 * (r >> 2) + 4 * h2 + (r & 3)), pair(o[db][r], o[db][r + 1]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (h2 == 0) __hip_atomic_store(place(run, DH), pair(m, l), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    partials_published(p.strict);
    __syncthreads();
    if (tid == 0) {
        s.ticket = take_ticket(&cut.counters[item], p.strict);
        if (s.ticket == (unsigned)(runs - 1)) __hip_atomic_store(&cut.counters[item], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s.ticket != (unsigned)(runs - 1) || !any) return;
    if (p.strict) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    auto load = [&](int r, int d, float &x, float &y) {
        const unsigned long long v = __hip_atomic_load(place(r, d), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        x = __uint_as_float((uint32_t)v);
        y = __uint_as_float((uint32_t)(v >> 32));
    };
    m = -INFINITY;
    l = 0.0f;
    o[0] = o[1] = floatx16{};
    // All loads of a run on their way at a time (the compiler would take them one by one: 5 us a run).
#pragma unroll 1
    for (int r = 0; r < runs; ++r) {
        float mr, lr;
        floatx16 x[2];
        load(r, DH, mr, lr);
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                float a, d;
                load(r, 32 * db + 8 * (e >> 2) + 4 * h2 + (e & 3), a, d);
                x[db][e] = a;
                x[db][e + 1] = d;
            }
        __builtin_amdgcn_sched_barrier(0);
        const float now = fmaxf(m, mr), keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - now), a = mr == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mr - now);
        m = now;
        l = fmaf(lr, a, l * keep);
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[db][e] = fmaf(x[db][e], a, o[db][e] * keep);
    }
    store(l);
}

// Requests with new rows of every number: those with up to eight rows of heads a K/V head (`slots` tokens) go token by token, the others in tiles.  A
// unit is a run of keys of a tile, or of a token, and a K/V head.  Up to 256 requests (`listed`) the units are numbered, tiles first, and runs are as long as it
// takes to keep the device busy; for more, the grid has places for as many as there could be.  Request b's tiles have places from
// query_start[b] * group / 128 + b on, which are enough for its rows, and more than all tiles of the requests before it need.
template <class T, int G, int MODE>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(const PagedAttn p, Runs tile_cut, Runs token_cut, int tile_places, int slots, int cus, int listed, const More<MODE> more) {
    union Shared {
        TileShared<T> tiles;
        TokenShared<G, 4> token;
    };
    __shared__ __align__(16) char smem[sizeof(Shared)];
    __shared__ Units tile_list, token_list;
    __shared__ int starts[kListed], lens[kListed], positions[kListed], runs_of_each[kListed];
    const int lane = threadIdx.x & 63, group = p.group.size;
    int tile_units = tile_places * p.n_kv * tile_cut.most, all = tile_units + p.batch * slots * p.n_kv * token_cut.most;
    if (listed) {
        int tiles[4], tokens[4], keys[4], rows[4], longest = 0;
        float tile_most = 0.0f, tile_work = 0.0f, token_work = 0.0f;  // (a prompt's tiles see one more than the other: the longest, and on average)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            tiles[j] = tokens[j] = keys[j] = rows[j] = 0;
            if (64 * j >= p.batch) continue;  // uniform
            if (64 * j + lane < p.batch) {
                const int start = p.query_start[64 * j + lane], end = p.query_start[64 * j + lane + 1], q_len = min(end, p.tokens) - start, kv_len = max(p.kv_lens[64 * j + lane], 0);
                starts[64 * j + lane] = start;
                lens[64 * j + lane] = rows[j] = q_len;
                positions[64 * j + lane] = kv_len - (end - start);
                if (start >= 0 && q_len > 0) {
                    keys[j] = max(keys_seen(p, kv_len, q_len > slots ? min(q_len, p.group.page(TILE_ROWS) + 2) : 1), 1);
                    if (q_len > slots) tiles[j] = (q_len * group + TILE_ROWS - 1) / TILE_ROWS;
                    else tokens[j] = q_len;
                }
            }
            tile_most += (float)tiles[j] * (float)keys[j];
            tile_work += (float)tiles[j] * ((float)keys[j] - (p.window > 0 ? 0.0f : 0.5f * (float)min(rows[j], keys[j])));
            token_work += (float)tokens[j] * (float)keys[j];
            longest = max(longest, keys[j]);
        }
        longest = (int)wave_minmax_u32<true>((unsigned)longest);
        // Runs for tiles as long as the longest, or as on average, which makes more of them: what takes less time, if that is the length of a run where all of them find a
        // place at once, and that of the average otherwise, and what a run takes besides (2048 rows from the first on, 16 heads, fp32: 124 us with the longest, 88; 3 x
        // 700 rows behind 300, 12 heads: 51 with the longest, 68).
        tile_work = wave_sum(tile_work) * p.n_kv;
        const float places = 2.0f * cus;
        auto time_of = [&](int run) {
            float units = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (64 * j < p.batch && tiles[j] > 0) units += (float)(tiles[j] * paged::runs_of(keys[j], run, tile_cut.most).runs);
            units = fmaxf(wave_sum(units) * p.n_kv, 1.0f);
            const float rounds = __builtin_ceilf(units / places);
            return rounds > 1.0f ? rounds * (tile_work / units + 192.0f) : (float)run + 192.0f;
        };
        const int by_longest = paged::run_for(wave_sum(tile_most) * p.n_kv, places, 256, longest, tile_cut.most);
        const int by_average = paged::run_for(tile_work, places, 256, longest, tile_cut.most);
        tile_cut.run = by_average != by_longest && time_of(by_average) < time_of(by_longest) ? by_average : by_longest;
        token_cut.run = paged::run_for(wave_sum(token_work) * p.n_kv, 2.0f * cus, 128, longest, token_cut.most);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (64 * j >= p.batch) continue;  // uniform
            const int runs = paged::runs_of(keys[j], tiles[j] > 0 ? tile_cut.run : token_cut.run, tiles[j] > 0 ? tile_cut.most : token_cut.most).runs;
            runs_of_each[64 * j + lane] = runs;
            tiles[j] *= runs * p.n_kv;
            tokens[j] *= runs * p.n_kv;
        }
        tile_units = tile_list.number(tiles, p.batch, lane);
        all = tile_units + token_list.number(tokens, p.batch, lane);
    }
    // Every second time in the opposite order, XCD by XCD: tiles come the longest first, so that who had the longest then has the shortest.
    for (int round = 0; round < (all + (int)gridDim.x - 1) / (int)gridDim.x; ++round) {
        const int turned = (int)gridDim.x - 8 - ((int)blockIdx.x & ~7) + ((int)blockIdx.x & 7);
        const int unit = round * (int)gridDim.x + ((round & 1) && gridDim.x % 8 == 0 ? turned : (int)blockIdx.x);
        if (unit >= all) continue;
        __syncthreads();  // the numbers, and what the last unit left
        int at = unit, b, h, run, tile = -1, token = -1;
        if (listed) {
            if (at < tile_units) {
                // consecutive workgroups go round the XCDs; an XCD takes consecutive units, whose tiles share a head's K and V
                const int each = tile_units >> 3, rest = tile_units & 7, xcd = at & 7;
                at = xcd * each + min(xcd, rest) + (at >> 3);
                b = tile_list.entry(at, lane);
                const int q_len = lens[b], n = (q_len * group + TILE_ROWS - 1) / TILE_ROWS;
                const int runs = runs_of_each[b];
                const int place = at / runs;
                run = at - place * runs;
                h = place / n;
                tile = n - 1 - (place - h * n);
            } else {
                at -= tile_units;
                b = token_list.entry(at, lane);
                const int runs = runs_of_each[b];
                token = at / (runs * p.n_kv);
                at -= token * runs * p.n_kv;
                run = at / p.n_kv;
                h = at - run * p.n_kv;
            }
        } else if (at < tile_units) {
            run = at % tile_cut.most;
            at /= tile_cut.most;
            h = at / tile_places;
            const int place = tile_places - 1 - (at - h * tile_places);
            b = -1;
            for (int i = 0; i < p.batch; i += 64) b += __popcll(__ballot(i + lane < p.batch && p.query_start[i + lane] * group / TILE_ROWS + i + lane <= place));
            if (b < 0) continue;
            tile = place - p.query_start[b] * group / TILE_ROWS - b;
        } else {
            at -= tile_units;
            run = at % token_cut.most;
            at /= token_cut.most;
            h = at % p.n_kv;
            at /= p.n_kv;
            b = at / slots;
            token = at - b * slots;
        }
        // (the rows that the call has of the request, which may have more: positions are theirs)
        const int start = listed ? starts[b] : p.query_start[b], q_len = listed ? lens[b] : min(p.query_start[b + 1], p.tokens) - start;
        const int pos_first = listed ? positions[b] : max(p.kv_lens[b], 0) - (p.query_start[b + 1] - start);
        if (start < 0) continue;
        if (token < 0) {
            if (q_len <= slots || tile < 0 || tile * TILE_ROWS >= q_len * group) continue;
            const int item = (start * group / TILE_ROWS + b + tile) * p.n_kv + h;
            tile_run<T>(p, more, *reinterpret_cast<TileShared<T> *>(smem), tile_cut, b, TileOf<MODE>{start, q_len, pos_first}, h, tile * TILE_ROWS, run, item);
        } else {
            if (token >= q_len || q_len > slots) continue;
            token_run<T, G, 4, 4>(p, more, *reinterpret_cast<TokenShared<G, 4> *>(smem), token_cut, start + token, b, pos_first + token, h, h * group, group, run,
                                  (b * slots + token) * p.n_kv + h);
        }
    }
}

// `scratch` bytes from `space` on are for partial results.
template <class T, int G, int MODE>
int32_t tokens_go(agpu_ctx *ctx, const PagedAttn &p, int64_t longest, const More<MODE> &more, char *space, size_t scratch) {
    const int64_t items = (int64_t)p.tokens * p.n_kv * ceil_div(p.n_heads / p.n_kv, G), places = 6 * ctx->num_cus;
    constexpr int part = G * (DH + 2), least = 128;
    // Where all the runs there could be find place at once, there is nothing to be counted: that takes 1.8 us (1 token of 12 heads, 777 keys: 10.0 / 8.2).
    const bool few = items * ((longest + least - 1) / least) <= places, listed = !few && p.tokens <= kListed;
    const int most = paged::most_runs(items, longest, few || listed ? least : 1024, part * sizeof(float), scratch / 2, ctx->n_counters - 1);
    const Runs cut = {few ? least : 1024, most, reinterpret_cast<float *>(space), part, ctx->counters};
    hipLaunchKernelGGL((paged_tokens_kernel<T, G, 4, 4, MODE>), dim3((unsigned)std::min<int64_t>(items * most, places)), dim3(256), 0, ctx->stream, p, cut,
                       2.0f * ctx->num_cus, least, (int)listed, more);
    return AGPU_LAUNCH_CHECK(ctx, "paged_tokens_kernel");
}
template <class T, int G, int MODE>
int32_t rows_go(agpu_ctx *ctx, const PagedAttn &p, int64_t longest, const More<MODE> &more, char *space, size_t scratch) {
    const int group = p.n_heads / p.n_kv, slots = 8 / group;  // up to eight rows: token by token
    const int tile_places = (int)((int64_t)p.tokens * group / TILE_ROWS) + p.batch;
    const int64_t tiles = (int64_t)tile_places * p.n_kv, tokens = (int64_t)p.batch * slots * p.n_kv;
    constexpr int tile_part = TILE_ROWS * (DH + 2), token_part = G * (DH + 2);
    const size_t for_tiles = scratch / 4 * 3;  // the rest for tokens, and half of the tickets each
    const int64_t tickets = (ctx->n_counters - 1) / 2;
    const bool listed = p.batch <= kListed;
    const int tile_most = paged::most_runs(tiles, longest, listed ? 256 : 2048, tile_part * sizeof(float), for_tiles, tickets);
    const int token_most = paged::most_runs(tokens, longest, listed ? 128 : 1024, token_part * sizeof(float), scratch - for_tiles, tickets);
    const Runs tile_cut = {2048, tile_most, reinterpret_cast<float *>(space), tile_part, ctx->counters};
    const Runs token_cut = {1024, token_most, reinterpret_cast<float *>(space + for_tiles), token_part, ctx->counters + tickets};
    const int64_t units = tiles * tile_most + tokens * token_most;
    if (units > INT32_MAX) return agpu_fail(ctx, AGPU_ERR_UNSUPPORTED, "paged_attention: %d tokens of %d requests are too many", p.tokens, p.batch);
    hipLaunchKernelGGL((paged_rows_kernel<T, G, MODE>), dim3((unsigned)std::min<int64_t>(units, 2 * ctx->num_cus)), dim3(256), 0, ctx->stream, p, tile_cut, token_cut, tile_places,
                       slots, ctx->num_cus, (int)listed, more);
    return AGPU_LAUNCH_CHECK(ctx, "paged_rows_kernel");
}
template <class T, int MODE>
int32_t attention_go(agpu_ctx *ctx, const PagedAttn &p, int64_t longest, const More<MODE> &more, char *space, size_t scratch) {
    const int g = p.n_heads / p.n_kv;
    auto go = [&](auto heads) {
        constexpr int G = decltype(heads)::value;
        return p.tokens <= p.batch ? tokens_go<T, G>(ctx, p, longest, more, space, scratch) : rows_go<T, G>(ctx, p, longest, more, space, scratch);
    };
    return g == 1 ? go(std::integral_constant<int, 1>{}) : g == 2 ? go(std::integral_constant<int, 2>{}) : g <= 4 ? go(std::integral_constant<int, 4>{}) : go(std::integral_constant<int, 8>{});
}
inline PagedAttn paged_attn(const float *q, int64_t q_row, int64_t q_head, const void *k, const void *v, int64_t k_page, int64_t v_page, const int32_t *tables,
                            const int32_t *kv_lens, const int32_t *query_start, float *o, int32_t tokens, int32_t batch, int32_t n_heads, int32_t n_kv_heads, int32_t n_pages,
                            int32_t page_size, int32_t width, int32_t window, int32_t sinks, int strict) {
    PagedAttn p{};
    p.q = q; p.q_row = q_row; p.q_head = q_head;
    p.k = k; p.v = v; p.k_page = k_page; p.v_page = v_page;
    p.tables = tables; p.kv_lens = kv_lens; p.query_start = query_start; p.o = o;
    p.tokens = tokens; p.batch = batch; p.n_heads = n_heads; p.n_kv = n_kv_heads; p.n_pages = n_pages;
    p.width = width; p.held = width * page_size; p.window = window; p.sinks = sinks;
    p.div = PageDiv::of(page_size);
    p.group = PageDiv::of(n_heads / n_kv_heads);
    p.strict = strict;
    return p;
}
// go(the cache's type)
template <class F>
int32_t of_type(int32_t cache_type, F go) {
    return cache_type == AGPU_CACHE_F32 ? go(F32{}) : cache_type == AGPU_CACHE_F16 ? go(F16{}) : go(BF16{});
}

}  // namespace
