// Attention of requests that begin alike, d_head = 64: o = softmax(q k / 8) v over the keys of a prefix, which lies in the cache once, and of each request's own pages behind
// it.  Two launches:
//   paged_prefix_kernel   the rows of all requests behind a prefix are rows of one product with its keys.  It leaves o, m and l (sum of weights 2^(s - m) times v, its unit,
//                         and their sum) of each row, in runs of keys.  Up to 128 rows of heads: wave_run, below.  More: tile_run, whose four waves share what is laid out of
//                         K and V (6 chunks of up to 150 rows, 16 heads, fp32, 1800 keys 50 us; by waves of their own 71.  Over 16-bit caches there is nothing to lay out,
//                         and both take the same).
//   paged_tokens_kernel, paged_rows_kernel (paged_kernels.h)   each request's own pages, as in paged_attention; what a row has seen of its prefix counts as keys of its own.
// What bounds it: 64 requests of 100 own keys on average, 25 heads, bf16, behind 4000 keys take 33 us, of which the bytes of K and V, each read once, are 13.  The prefix's
// half is 17: 1 until all workgroups are there, 3 until a tile's rows are known (requests counted by prefix, runs cut, rows listed: loads, sums and divisions that wait for one
// another), 8 to 10 for 3.5 tiles of 32 keys a wave (2900 cycles one after the other: 800 from LDS to operands, 400 the next tile's request, 460 products, 420 softmax, 900 weights and
// products; the SIMDs issue a third of the time), 1.5 to join the waves, 0.5 for the last stores.  (Two waves a SIMD, as both ways share one budget of registers; over
// fp32 20 of them are spilled.  Runs go by the prefix's length: a window leaves them as they are, and those that it hides are empty.)  The other half is what paged_attention takes for the own pages (15) and 2 for the prefix's runs.
#include "paged_kernels.h"

namespace {

// The requests' rows, counted by prefix, and the places of a tile's rows.
struct PrefixShared {
    int rows[paged::kMaxPrefixes], len[paged::kMaxPrefixes];
    int token[TILE_ROWS], pos[TILE_ROWS];
    int wave_rows[4], pos0[4], pos1[4];
    float m[4][32];
};

// The rows that the call has of a request: the prefix, how many, the first, and where it is among own positions.
struct Behind {
    int g, count, start, pos;
    __device__ __forceinline__ Behind(const PagedAttn &p, const More<PREFIX> &more, int b) {
        const int at = min(b, p.batch - 1);  // (what is loaded is loaded together)
        g = more.of[at];
        start = p.query_start ? p.query_start[at] : at;
        const int end = p.query_start ? p.query_start[at + 1] : at + 1;
        pos = min(max(p.kv_lens[at], 0), (int)paged::kMaxPositions) - (end - start);
        count = min(end, p.tokens) - start;
        if (b >= p.batch || start < 0 || count < 0 || (unsigned)g >= (unsigned)more.n_prefix) count = 0;
    }
};

// Straight to memory: what the next launch reads is not left for the end of this one (64 requests 18.7 us, 18.0).
__device__ __forceinline__ void store2_through(float *to, float a, float b) {
    __hip_atomic_store(reinterpret_cast<unsigned long long *>(to), (unsigned long long)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store4_through(float *to, const float4 &v) {
    store2_through(to, v.x, v.y);
    store2_through(to + 2, v.z, v.w);
}

// ---- few rows: a wave's 32 rows over tiles of keys of its own -------------------------------------

constexpr int kJoinRow = DH + 4;  // floats of a row of o in LDS
template <class T>
struct WaveTile {
    static constexpr int kRow = 64 * 16 / T::EL;  // bytes of a row of K or V
    char k[TILE_KEYS * kRow], v[TILE_KEYS * kRow];  // rows as they are in the cache, their 16-byte pieces in an order by which what is read at a time lies in different banks
    long long at[2][2][2 * TILE_KEYS];              // where the rows of K and of V of two tiles begin, in bytes; by turns for this pair and the next one
};
template <class T>
union WaveShared {
    WaveTile<T> tile[4];
    struct {
        float o[4][32][kJoinRow], m[4][32], l[4][32];
    } join;
};

// 16 bytes a lane from `from` into LDS, one lane behind the other from `to` (uniform) on; nothing waits for them here.
__device__ __forceinline__ void load_to_lds(uint32_t to, const char *from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}

// What 32 rows see of tiles of 32 keys: number i is the keys from first_key + i * stride on, up to `hi`.  This lane's row is at `pos`, all rows at pos0 .. pos1.  Without a
// window id and off are the first two tiles': the page of key first_key + stride * (lane / 32) + lane % 32, and where on it.  A tile goes from the
// cache to LDS by itself, whole lines at a time, while the one before it is worked on, whose operands are in registers by then: no barrier, and no wave waits for another.  (Rows
// straight into operand registers are reads of 32 bytes from each of 32 lines: 8 requests behind 500 keys, fp32, 13.3 us, 9.8 this way.)
template <class T>
__device__ __forceinline__ void wave_run(const PagedAttn &p, WaveTile<T> &s, int g, int h, const paged::TileKeys &keys, int pos, int pos0, int pos1, const float *q_row,
                                         int first_key, int stride, int hi, int id, int off, float &m, float &l, floatx16 (&o)[2]) {
    constexpr int KP = Tiles<T>::KP, QP = Tiles<T>::QP, kBytes = 16 / T::EL, kRow = WaveTile<T>::kRow, PIECES = kRow / 16, LOADS = TILE_KEYS * kRow / 1024;
    const int lane = threadIdx.x & 63, c = lane & 31, h2 = lane >> 5, gap = keys.gap;
    const paged::RowKeys see = paged::row_keys(keys, pos, p.window, p.sinks);
    const int low = paged::row_keys(keys, pos1, p.window, p.sinks).low;
    const int *table = p.tables + (size_t)g * p.width;
    const char *const kb = static_cast<const char *>(p.k), *const vb = static_cast<const char *>(p.v);
    const int tiles = first_key < hi ? (hi - first_key + stride - 1) / stride : 0;
    auto look_up = [&](int i) {  // tiles i and i + 1, one a half wave
        const int v = first_key + (i + h2) * stride + c;
        id = -1;
        off = 0;
        if (i + h2 < tiles && v < hi) {
            const int j = keys.key(v), page = p.div.page(j);
            id = table[page];
            off = j - page * p.div.size;
        }
    };
    if (p.window > 0) look_up(0);
    else if (first_key + h2 * stride + c >= hi) id = -1;
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
    // Where piece `at` of a key's row lies in LDS.
    auto k_place = [&](int key, int at) { return key * kRow + 16 * (at ^ (key & (PIECES - 1))); };
    auto v_turn = [&](int key) { return PIECES == 16 ? (key >> 2 & 1) << 3 : ((key & 2) ^ (key >> 2 & 1)) << 1; };  // (of 16-bit rows as tile_v_at says)
    const uint32_t lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(size_t)(__attribute__((address_space(3))) char *)(s.k));
    uint64_t held = 0, held_next = 0;  // which keys of a pair of tiles are there
    // Where the rows of tiles i and i + 1 are, which have been looked up; the two behind them are now, so that who waits for a tile has waited for that too.
    auto prepare = [&](int i) {
        const bool ok = (unsigned)id < (unsigned)p.n_pages;
        const long long row = (long long)(h * p.div.size + off) * DH;
        s.at[i >> 1 & 1][0][lane] = ok ? (id * p.k_page + row) * kBytes : 0;
        s.at[i >> 1 & 1][1][lane] = ok ? (id * p.v_page + row) * kBytes : 0;
        held_next = __ballot(ok);
        look_up(i + 2);
    };
    // Tile i on its way.  `from`, where this lane's rows begin, is read together, as nothing goes past the loads, which are written out.
    struct From {
        long long at[2][LOADS];
    };
    const int slot = lane % PIECES;
    auto places = [&](int i) {
        From f;
#pragma unroll
        for (int n = 0; n < 2 * LOADS; ++n) f.at[n / LOADS][n % LOADS] = s.at[i >> 1 & 1][n / LOADS][TILE_KEYS * (i & 1) + n % LOADS * (64 / PIECES) + lane / PIECES];
        return f;
    };
    auto request = [&](const From &f) {
#pragma unroll
        for (int n = 0; n < 2 * LOADS; ++n) {
            const int key = n % LOADS * (64 / PIECES) + lane / PIECES;
            load_to_lds(lds + 1024 * n, n < LOADS ? kb + f.at[0][n % LOADS] + 16 * (slot ^ (key & (PIECES - 1))) : vb + f.at[1][n % LOADS] + 16 * (slot ^ v_turn(key)));
        }
    };
    const int turned = tile_v_at(4 * h2 + ((lane & 15) >> 2), c >> 4) + 8 * (lane & 3);
    m = -INFINITY;
    l = 0.0f;
    o[0] = o[1] = floatx16{};
    if (tiles > 0) {
        prepare(0);
        request(places(0));
    }
    for (int i = 0; i < tiles; ++i) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if ((i & 1) == 0) held = held_next;
        const uint32_t there = (uint32_t)(held >> (32 * (i & 1)));
        Staged<T> sk[4], sv[2][2];  // K: of key c the elements 16 ds + 8 h2 ..; V: of dimension 32 db + c the keys 16 st + 8 (e / 4) + 4 h2 + e mod 4
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) {
            if constexpr (PIECES == 16) {
                const float4 a = *reinterpret_cast<const float4 *>(s.k + k_place(c, 4 * ds + 2 * h2)), d = *reinterpret_cast<const float4 *>(s.k + k_place(c, 4 * ds + 2 * h2 + 1));
                const float y[8] = {a.x, a.y, a.z, a.w, d.x, d.y, d.z, d.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) sk[ds].x[e] = y[e];
            } else {
                sk[ds].row(s.k + k_place(c, 2 * ds + h2));
            }
        }
        auto read_v = [&] {
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int db = 0; db < 2; ++db) {
                    if constexpr (PIECES == 16) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            sv[st][db].x[e] = *reinterpret_cast<const float *>(s.v + (16 * st + 8 * (e >> 2) + 4 * h2 + (e & 3)) * kRow + 16 * ((8 * db + (c >> 2)) ^ (h2 << 3)) + 4 * (c & 3));
                    } else {
                        typedef short four __attribute__((ext_vector_type(4)));
                        typedef __attribute__((address_space(3))) four *in_lds;
                        const char *const at = s.v + (turned ^ (64 * db)) + 2048 * st;
                        const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((in_lds)at)), d = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((in_lds)(at + 1024)));
                        sv[st][db].x[0] = a.x; sv[st][db].x[1] = a.y; sv[st][db].x[2] = d.x; sv[st][db].x[3] = d.y;
                    }
                }
        };
        read_v();
        if (there != 0xffffffffu && !(there >> c & 1))  // zeros instead of what is not there (of V, that has no weight)
#pragma unroll
            for (int ds = 0; ds < 4; ++ds) sk[ds].clear();
        // V with something infinite or no number in it goes in as zeros, and is added below for the rows that see it.
        uint32_t odd_k = 0, odd_v = 0;
        bool odd = false;
        if constexpr (PIECES == 16) {
#pragma unroll
            for (int n = 0; n < 4; ++n) odd |= sv[n >> 1][n & 1].odd();
        } else {  // (a number of 2^65 or more, 2^9 in f16, is looked at more closely)
            uint32_t two = 0;
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) two |= sv[n >> 1][n & 1].x[e] & sv[n >> 1][n & 1].x[e] << 1;
            odd = (two & 0x40004000u) != 0;
        }
        const long long k_at = s.at[i >> 1 & 1][0][TILE_KEYS * (i & 1) + c], v_at = s.at[i >> 1 & 1][1][TILE_KEYS * (i & 1) + c];  // for the odd ones
        if (__builtin_expect(__any(odd), 0)) {
            bool in_v = false;
#pragma unroll
            for (int n = 0; n < 4; ++n) {  // the rows themselves
                Staged<T> x;
                char *const at = s.v + c * kRow + (kRow / 8) * (4 * h2 + n);
                x.row(at);
                in_v |= x.odd();
                x.clean();
                if constexpr (PIECES == 16) {
                    *reinterpret_cast<float4 *>(at) = make_float4(x.x[0], x.x[1], x.x[2], x.x[3]);
                    *reinterpret_cast<float4 *>(at + 16) = make_float4(x.x[4], x.x[5], x.x[6], x.x[7]);
                } else {
                    *reinterpret_cast<uint4 *>(at) = make_uint4(x.x[0], x.x[1], x.x[2], x.x[3]);
                }
            }
            const uint64_t v2 = __ballot(in_v);
            odd_v = ((uint32_t)v2 | (uint32_t)(v2 >> 32)) & there;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            read_v();
        }
        if (i + 1 < tiles) {
            const From next = places(i + 1);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what is read of this tile is in registers
            request(next);
        }
        uint4 k[4][KP];
#pragma unroll
        for (int ds = 0; ds < 4; ++ds) sk[ds].pieces(k[ds]);
        const int v0 = first_key + i * stride;
        auto row_of = [](long long at, int kk) {  // key kk's
            return (size_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)at, kk) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(at >> 32), kk) << 32);
        };
        floatx16 x = {};
#pragma unroll
        for (int level = QP - 1; level >= 0; --level)
#pragma unroll
            for (int ds = 0; ds < 4; ++ds)
#pragma unroll
                for (int kp = KP - 1; kp >= 0; --kp)
                    if (level - kp >= 0 && level - kp < QP) x = Tiles<T>::mfma(k[ds][kp], q[ds][level - kp], x);
        if ((i & 1) == 0 && i + 2 < tiles) prepare(i + 2);
        // only tiles at the ends of what rows see hide anything (uniform)
        const bool whole = there == 0xffffffffu && v0 + TILE_KEYS - 1 <= pos0 - gap && (v0 > low || v0 + TILE_KEYS <= see.first);
        auto in_sight = [&] {  // of this row, one bit a key
            auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; };  // bits 0 .. n - 1
            return there & below(see.last + 1 - v0) & (~below(see.low + 1 - v0) | below(see.first - v0));
        };
        auto hide = [&] {
            if (whole) return;
            const uint32_t seen = in_sight() >> (4 * h2);
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = seen >> (8 * (r >> 2) + (r & 3)) & 1 ? x[r] : -INFINITY;
        };
        auto highest = [&] {  // no number, if one of them is none
            float top = x[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = __builtin_elementwise_maximum(top, x[r]);
            return top;
        };
        hide();
        float top = highest();
        if (__builtin_expect(__any(!(top < INFINITY)), 0)) {
            // Something infinite or no number among what rows see: scores of keys that have it in K are formed in fp32 (others' are what they are).
            bool in_k = false;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                Staged<T> y;
                y.row(kb + k_at + (kRow / 8) * (4 * h2 + n));
                in_k |= y.clean() != 0;
            }
            const uint64_t k2 = __ballot(in_k);
            odd_k = ((uint32_t)k2 | (uint32_t)(k2 >> 32)) & there;
#pragma unroll 1
            for (int kk = 0; kk < TILE_KEYS; ++kk) {
                if (!(odd_k >> kk & 1)) continue;
                const size_t at = row_of(k_at, kk);
                float d = 0.0f;
#pragma unroll 1
                for (int e = 0; e < 32; ++e) d = fmaf(q_row[32 * h2 + e] * kQueryScale, T::one(kb + at, 32 * h2 + e), d);
                d = sum_of_halves(d) / unit;
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = 8 * (r >> 2) + 4 * h2 + (r & 3) == kk ? d : x[r];
            }
            hide();
            top = x[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
        }
        top = max_of_halves(top) * unit;
        // Weights grow to 2^6 before a row is rescaled, but not beside values from 2^91 on, as in tile_run.
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
            x[r] = __builtin_amdgcn_exp2f(QP == 2 ? fmaf(x[r], unit, -ref) : x[r] - ref);
            sum += x[r];
        }
        l += sum;
        uint4 w[2][QP], v[2][2][KP];
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[8 * st + e] * Tiles<T>::UP;
            pieces_of(y, w[st]);
#pragma unroll
            for (int db = 0; db < 2; ++db) sv[st][db].pieces(v[st][db]);
        }
#pragma unroll
        for (int level = QP - 1; level >= 0; --level)
#pragma unroll
            for (int kp = KP - 1; kp >= 0; --kp)
                if (level - kp >= 0 && level - kp < QP)
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int db = 0; db < 2; ++db) o[db] = Tiles<T>::mfma(v[st][db][kp], w[st][level - kp], o[db]);
        if (__builtin_expect(odd_v != 0, 0))
#pragma unroll 1
            for (int kk = 0; kk < TILE_KEYS; ++kk) {
                if (!(odd_v >> kk & 1)) continue;
                const bool sees = see.sees(v0 + kk);
                float weight = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) weight = 8 * (r >> 2) + 4 * h2 + (r & 3) == kk ? x[r] : weight;
                weight = sum_of_halves(weight);  // (one of them is zero)
                const size_t at = row_of(v_at, kk);
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
}

constexpr int kWaveRows = 128;  // more go through tile_run

// p.tables, p.width and p.held are the prefixes'.
template <class T>
__global__ __launch_bounds__(256, 2) void paged_prefix_kernel(const PagedAttn p, Runs cut, int cus, const More<PREFIX> more) {
    __shared__ union {
        TileShared<T> tile;
        WaveShared<T> wave;
    } u;
    __shared__ Units list;
    __shared__ PrefixShared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = p.group.size;
    const Behind mine(p, more, tid);
    if (tid < more.n_prefix) {
        s.len[tid] = more.len(tid);
        s.rows[tid] = 0;
    }
    __syncthreads();
    if (mine.count > 0) atomicAdd(&s.rows[mine.g], mine.count);
    for (int b = tid + 256; b < p.batch; b += 256) {
        const Behind other(p, more, b);
        if (other.count > 0) atomicAdd(&s.rows[other.g], other.count);
    }
    __syncthreads();
    auto rows_behind = [&](int g) { return min(max(s.rows[g], 0), p.tokens) * group; };  // (query_starts that overlap may count to more than there are, or than an int holds)
    int tiles[4], keys[4], longest = 0;
    float work = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        tiles[j] = keys[j] = 0;
        if (64 * j >= more.n_prefix) continue;  // uniform
        const int g = 64 * j + lane;
        if (g < more.n_prefix) {
            keys[j] = s.len[g];
            tiles[j] = keys[j] > 0 ? (rows_behind(g) + TILE_ROWS - 1) / TILE_ROWS : 0;
        }
        work += (float)tiles[j] * (float)keys[j];
        longest = max(longest, keys[j]);
    }
    cut.run = paged::run_for(wave_sum(work) * p.n_kv, 2.0f * cus, 128, (int)wave_minmax_u32<true>((unsigned)longest), cut.most);
    if (blockIdx.x == 0) {
        auto leave = [&](int b, const Behind &r) {
            const int len = (unsigned)r.g < (unsigned)more.n_prefix ? s.len[r.g] : 0;
            if (b < p.batch) more.before[b] = len > 0 ? paged::runs_of(len, cut.run, cut.most).runs : 0;
        };
        leave(tid, mine);
        for (int b = tid + 256; b < p.batch; b += 256) leave(b, Behind(p, more, b));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (64 * j < more.n_prefix) tiles[j] *= paged::runs_of(keys[j], cut.run, cut.most).runs * p.n_kv;
    const int all = list.number(tiles, more.n_prefix, lane);
    for (int unit = blockIdx.x; unit < all; unit += gridDim.x) {
        __syncthreads();  // the numbers, and what the last unit left
        int at = unit;
        const int g = __builtin_amdgcn_readfirstlane(list.entry(at, lane)), rows = __builtin_amdgcn_readfirstlane(rows_behind(g)), n = (rows + TILE_ROWS - 1) / TILE_ROWS;
        const int len = __builtin_amdgcn_readfirstlane(s.len[g]);
        const paged::RunsOf cuts = paged::runs_of(len, cut.run, cut.most);
        const int place = at / n, first_row = (at - place * n) * TILE_ROWS, last_row = min(first_row + TILE_ROWS, rows) - 1;
        const int h = place / cuts.runs, run = place - h * cuts.runs, lo = run * cuts.keys;
        // Few rows: waves for every 32 of them, and as many for each as there are; these take the keys of a run by turns.
        const int sets = last_row - first_row < 32 ? 1 : last_row - first_row < 64 ? 2 : 4, turns = 4 / sets, first_key = lo + TILE_KEYS * (wave / sets);
        int id = -1, off = 0;
        if (rows <= kWaveRows && first_key + TILE_KEYS * turns * (lane >> 5) + (lane & 31) < len) {  // (of use where no window moves the keys)
            const int j = first_key + TILE_KEYS * turns * (lane >> 5) + (lane & 31), page = p.div.page(j);
            id = p.tables[(size_t)g * p.width + page];
            off = j - page * p.div.size;
        }
        // which tokens the tile's rows are of: the prefix's tokens in the order of the requests
        const int first = p.group.page(first_row), last = p.group.page(last_row);
        int before = 0, pos0 = INT32_MAX, pos1 = INT32_MIN;
        auto list_rows = [&](const Behind &r) {
            const int count = r.g == g ? r.count : 0, upto = wave_running_sum(count);
            if (lane == 63) s.wave_rows[wave] = upto;
            __syncthreads();
            int at = before + upto - count;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (w < wave) at += s.wave_rows[w];
                before += s.wave_rows[w];
            }
            // rows from .. to - 1 of this thread's request are the tile's; its own thread writes them where they are few, and its wave where they are many
            const int from = max(first - at, 0), to = min(count, last + 1 - at);
            if (to > from) {
                pos0 = min(pos0, len + r.pos + from);
                pos1 = max(pos1, len + r.pos + to - 1);
            }
            constexpr int kFew = 4;
#pragma unroll
            for (int e = 0; e < kFew; ++e) {
                const int i = from + e;
                if (to - from <= kFew && i < to) s.token[at + i - first] = r.start + i, s.pos[at + i - first] = len + r.pos + i;
            }
            for (uint64_t many = __ballot(to - from > kFew); many != 0; many &= many - 1) {  // uniform
                const int who = __builtin_ctzll(many), at_w = __builtin_amdgcn_readlane(at, who), to_w = __builtin_amdgcn_readlane(to, who);
                const int start_w = __builtin_amdgcn_readlane(r.start, who), pos_w = __builtin_amdgcn_readlane(r.pos, who);
                for (int i = __builtin_amdgcn_readlane(from, who) + lane; i < to_w; i += 64) s.token[at_w + i - first] = start_w + i, s.pos[at_w + i - first] = len + pos_w + i;
            }
        };
        list_rows(mine);
        for (int b = 256; b < p.batch && before <= last; b += 256) {
            __syncthreads();
            list_rows(Behind(p, more, b + tid));
        }
        constexpr uint32_t up = 0x80000000u;  // (numbers of either sign in the order of unsigned ones)
        pos0 = (int)(wave_minmax_u32<false>((uint32_t)pos0 ^ up) ^ up);
        pos1 = (int)(wave_minmax_u32<true>((uint32_t)pos1 ^ up) ^ up);
        if (lane == 0) s.pos0[wave] = pos0, s.pos1[wave] = pos1;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) pos0 = min(pos0, s.pos0[w]), pos1 = max(pos1, s.pos1[w]);
        pos0 = __builtin_amdgcn_readfirstlane(pos0), pos1 = __builtin_amdgcn_readfirstlane(pos1);
        if (rows > kWaveRows) {
            tile_run<T>(p, more, u.tile, cut, g, TileOf<PREFIX>{s.token, s.pos, first, min(s.rows[g], p.tokens), pos0, pos1}, h, first_row, run, 0);
            continue;
        }
        const int c = lane & 31, h2 = lane >> 5;
        const int row = min(first_row + 32 * (wave % sets) + c, last_row), token = p.group.page(row), head = h * group + (row - token * group);
        const paged::TileKeys seen = paged::tile_keys(pos0, pos1, len, p.window, p.sinks);
        float m, l;
        floatx16 o[2];
        wave_run<T>(p, u.wave.tile[wave], g, h, seen, s.pos[token - first], pos0, pos1, p.q + (size_t)s.token[token - first] * p.q_row + (size_t)head * p.q_head,
                    first_key, TILE_KEYS * turns, min(seen.count, lo + cuts.keys), id, off, m, l, o);
        // The waves of the same rows together, in units of the largest maximum.
        if (h2 == 0) s.m[wave][c] = m;
        __syncthreads();
        float top = m;
        for (int k = 1; k < turns; ++k) top = fmaxf(top, s.m[(wave + sets * k) & 3][c]);
        const float f = (m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top)) / Tiles<T>::UP;
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<float4 *>(&u.wave.join.o[wave][c][32 * db + 2 * r + 4 * h2]) = make_float4(o[db][r] * f, o[db][r + 1] * f, o[db][r + 2] * f, o[db][r + 3] * f);
        if (h2 == 0) u.wave.join.m[wave][c] = top, u.wave.join.l[wave][c] = l * (f * Tiles<T>::UP);
        __syncthreads();
        const size_t rows_all = (size_t)p.tokens * p.n_heads;
        auto finish = [&](auto waves) {  // four dimensions of a row a thread, four waves' rows at most
            constexpr int TURNS = decltype(waves)::value, SETS = 4 / TURNS;
#pragma unroll
            for (int n = 0; n < 2 * SETS; ++n) {
                const int at = 16 * n + (tid >> 4), set = n >> 1, d = 4 * (tid & 15);
                if (first_row + at > last_row) continue;
                const int token = p.group.page(first_row + at), head = h * group + (first_row + at - token * group);
                float4 all = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < TURNS; ++k) {
                    const float4 x = *reinterpret_cast<const float4 *>(&u.wave.join.o[set + SETS * k][at & 31][d]);
                    all = make_float4(all.x + x.x, all.y + x.y, all.z + x.z, all.w + x.w);
                    sum += u.wave.join.l[set + SETS * k][at & 31];
                }
                const size_t row_at = (size_t)s.token[token - first] * p.n_heads + head;
                store4_through((run == 0 ? more.first + row_at * DH : more.rest + ((run - 1) * rows_all + row_at) * DH) + d, all);
                if (d == 0) store2_through(&more.ml[run * rows_all + row_at].x, u.wave.join.m[set][at & 31], sum);
            }
        };
        if (turns == 4) finish(std::integral_constant<int, 4>{});
        else if (turns == 2) finish(std::integral_constant<int, 2>{});
        else finish(std::integral_constant<int, 1>{});
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
    // Scratch: how many runs there are before each request, (m, l) of the prefix's runs and o of those that the results have no place for, half of it at most; then the
    // partial results over own pages.
    const bool apart = (uintptr_t)o % 16 != 0;
    const paged::PrefixRuns room = paged::prefix_runs(batch, (int64_t)tokens * n_heads, (int64_t)prefix_width * page_size, apart, ctx->ws_bytes);
    if (room.most == 0) return agpu_fail(ctx, AGPU_ERR_WORKSPACE, "paged_attention_shared: %d rows of %d heads need a larger scratch", tokens, n_heads);
    More<PREFIX> pre{};
    pre.tables = prefix_tables; pre.lens = prefix_lens; pre.of = prefix_of; pre.n_prefix = n_prefix; pre.width = prefix_width; pre.held = prefix_width * page_size;
    pre.before = reinterpret_cast<int *>(ctx->workspace);
    pre.ml = reinterpret_cast<float2 *>(ctx->workspace + room.ml);
    pre.rest = reinterpret_cast<float *>(ctx->workspace + room.rest);
    pre.first = apart ? pre.rest + (int64_t)(room.most - 1) * tokens * n_heads * DH : o;
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
