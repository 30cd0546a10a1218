// The draw of the next tokens from rows of logits: temperature, top-k, top-p and min-p, and one given number of [0, 1) a row.
//   w_i = exp((x_i - max) / T); candidates ranked by x, the largest first, the lower index first among equals.
// Each filter keeps a first part of the ranking (the k first; those before which less than p of the k's sum lies; w >= min_p), so that what is kept is the
// shortest of the three parts, and all that the draw needs of it is its sum Z: the token is the first rank whose running sum exceeds u Z.
//
// Sums decide, next to borders, which token comes out, and there are tens of thousands of terms: weights are whole numbers, 2^45 for a weight of
// one at 50257 logits, from an exponential in 64-bit floats (off by 8e-14 of itself), and their sums are exact in any order.  (With fp32 exponentials a row
// of 50257 logits would go wrong about once in a thousand draws.)
//
// sample_rows_kernel, a workgroup a row, one launch, no scratch (50257 logits: top 40 of 1 row 13 us, 32 rows of all kinds 32, the nucleus of 256 rows 35, of
// which the read of 51 MB is 11).  Bound by the way of one row through one CU, whatever the number of rows.  Of its 63000 cycles, with a nucleus of 0.95 among 32
// rows, 5000 go by until there are logits, 14000 in a wave's pass (some 22 instructions a weight, 9 of them in 64 bits) and 10000 until the last wave is through, 4000 in
// the running sums, 4000 in the bins of the borders, 13000 in looking through all elements' bins for those, 3000 in putting what is in them in order, 4000 in its sums and
// 5000 in the filters and the draw.  Several workgroups a row and three launches were 22, 32 and 70 us.
//   general   One pass over the row adds up the weights in bins of 1/32 of an octave, each in units of its bin's middle (a polynomial of degree four is then exact to
//             8e-14), so that the largest logit need not be known before: 64 octaves fit, and the first 4096 elements say where they lie.  Which bin an element
//             went to stays in LDS.  From the bins' running sums follows in which bins the filters' borders lie, between which sums Z then is, and in which
//             bins the drawn rank can be: only what is in those, a few hundred elements, is gathered, put in order by counting, and searched.
//   top_k up to 256   The top_k-th largest of the threads' maxima is a bound that hardly more than top_k elements reach: the list is those.
// When the bins hold more than the list (thousands of equal logits, a large temperature), each border is looked for by itself, in the elements of
// its bin cut into 512 by the first bits in which their (value, index), which are never the same twice, differ, until a piece fits: three passes over the row for each border as a rule (64 rows at
// temperature 5 with a nucleus of 0.9 140 to 164 us, at temperature 2 97, rows of equal logits 302).
#include "agpu_internal.h"
#include "sampling.h"

#include <algorithm>

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 1024, SM_WAVES = SM_THREADS / 64;
constexpr int SM_BINS = 2048, SM_OCTAVE = 32;  // bins, and how many an octave has
constexpr int SM_LIST = 1024, SM_TOP_K = 256;  // (an element a thread)
constexpr int SM_PIECES = 512, SM_PIECE = 256;  // of a bin that does not fit: into how many it is cut, and what a piece may have
constexpr int SM_IDS = 56832;  // elements whose bins LDS has room for
constexpr int SM_AHEAD = 4;    // runs of four elements that a thread has on their way at a time
constexpr int kIndexBits = 20, kKeyBits = 52;  // n <= 2^20; of a value and its index
constexpr int kIdShift = 5;  // an element's bin is kept as that many bits further up, where 16 bits wrap as the bins do
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct SampleArgs {
    const float *logits, *u;
    const float *temperatures, *top_ps, *min_ps;
    const int *top_ks;
    float temperature, top_p, min_p;
    int top_k;
    int *tokens;
    int n, bits;  // a weight of one is 2^bits: sums of n weights stay below 2^62, and one below 2^51
};

// 2^f on [-1/2, 1/2], through 2^f at nine Chebyshev nodes and 1 at zero: off by 3.7e-14
__device__ __forceinline__ double exp2_part(double f) {
    double y = 1.0203115707778471e-07;
    y = fma(y, f, 1.3255224878668817e-06);
    y = fma(y, f, 1.5252686876393043e-05);
    y = fma(y, f, 1.5403455852453838e-04);
    y = fma(y, f, 1.3333558178986627e-03);
    y = fma(y, f, 9.618129159402558e-03);
    y = fma(y, f, 5.550410866476082e-02);
    y = fma(y, f, 2.402265069581299e-01);
    y = fma(y, f, 6.931471805599453e-01);
    return fma(y, f, 1.0);
}
__device__ __forceinline__ double exp2_wide(double t) {
    const double k = __builtin_rint(t);
    return __builtin_amdgcn_ldexp(exp2_part(t - k), (int)k);
}

// The bin of a logit and its weight in units of its bin: 32 log2 of it is t = (x - origin) per, its bin the whole number next to t, and its weight 2^f, f the rest / 32.
struct Scale {
    double per, origin, one;
    float low, high;  // what counts: within 48 octaves below the origin and 15 above it (NaN does not), 2017 bins of the 2048
    static constexpr int kNone = -48 * SM_OCTAVE - 8;  // a bin that nothing has
    __device__ __forceinline__ void set(double at, double temperature, int bits) {
        per = SM_OCTAVE * 1.4426950408889634 / temperature;
        origin = at;
        one = __builtin_bit_cast(double, 1ull << bits);  // 2^(bits - 1074)
        const double least = at - 48 * SM_OCTAVE / per, most = at + 15 * SM_OCTAVE / per;  // to the inside, whose ends a number may lie hundreds of octaves off
        low = (float)least;
        high = (float)most;
        if (low < least) low = key_value(order_key(low) + 1);
        if (high > most) high = key_value(order_key(high) - 1);
    }
    __device__ __forceinline__ bool counts(float x) const { return x >= low && x <= high; }
    static constexpr double kWhole = 0x1.8p52;  // added to it, a number's low bits are the whole number next to it
    // a b + c with c in scalar registers, where it stays (left to itself the compiler copies it into the result first)
    static __device__ __forceinline__ double fma_of(double a, double b, double c) {
        asm("v_fma_f64 %0, %1, %2, %3" : "=v"(a) : "v"(a), "v"(b), "s"(c));
        return a;
    }
    __device__ __forceinline__ int bin(float x, u64 &weight) const {
        const double fourth = 9.172562701824643e-09;
        const double d = (double)x - origin, v = fma(d, per, kWhole), f = fma(d, per, kWhole - v);
        // 2^(f / 32) for |f| <= 1/2: the series to the fifth power, that one through the fifth Chebyshev polynomial as the first and the third
        double y = fma_of(f, fourth, 1.6938633902808830e-06);
        y = fma_of(y, f, 2.3459619820224677e-04);
        y = fma_of(y, f, 2.1660849391722176e-02);
        y = fma(y, f, 1.0);
        weight = __builtin_bit_cast(u64, y * one);  // a denormal number, whose bits are the whole number that it was rounded to
        return (int)(uint32_t)__builtin_bit_cast(u64, v);
    }
    __device__ __forceinline__ int bin(float x) const { return (int)(uint32_t)__builtin_bit_cast(u64, fma((double)x - origin, per, kWhole)); }
    __device__ __forceinline__ u64 weight(float x) const {
        u64 w;
        bin(x, w);
        return w;
    }
};
// a sum of weights in bin j, `scale` = 2^(-j / 32), in units of bin 0: never smaller for a larger sum, and bin 0's as it is
__device__ __forceinline__ u64 in_units(u64 sum, double scale) { return scale == 1.0 ? sum : (u64)__builtin_rint((double)sum * scale); }
__device__ __forceinline__ double units(int j) { return exp2_wide(-(double)j / SM_OCTAVE); }

__device__ __forceinline__ u64 composite(float x, int i) { return (u64)order_key(x) << kIndexBits | (u64)((1 << kIndexBits) - 1 - i); }
__device__ __forceinline__ float value_of(u64 c) { return key_value((uint32_t)(c >> kIndexBits)); }
__device__ __forceinline__ int index_of(u64 c) { return (1 << kIndexBits) - 1 - (int)(c & ((1 << kIndexBits) - 1)); }

template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 v) {
    return (u64)dpp_move_u32<CTRL, ROWS>(0, (uint32_t)(v >> 32)) << 32 | dpp_move_u32<CTRL, ROWS>(0, (uint32_t)v);
}
// Sum over the lanes up to this one: row_shr 1, 2, 4, 8, then row_bcast 15 and 31.
__device__ __forceinline__ u64 sum_up_to(u64 v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    return v + moved<0x143, 0xc>(v);
}

struct Shared {
    u64 sum[SM_BINS];
    uint32_t count[SM_BINS];
    uint16_t id[SM_IDS];
    u64 list[SM_LIST], ranked[SM_LIST];  // elements in any order, and in that of the ranking; then list: running sums
    int place[SM_LIST];
    u64 wave_sum[SM_WAVES], answer_sum, kept_of_min_p, piece_sum, least, most;
    uint32_t wave_count[SM_WAVES], answer_index, piece_count;
    float wave_top[SM_WAVES];
    uint32_t top[SM_THREADS];
    int hit[2], from[4], to[4], fill, piece;
};

// share times sum, 0 < share < 1, cut off, and whether nothing was: sums have more bits than 64-bit floats, in which a border between equal weights would be missed.
__device__ __forceinline__ u64 mostof(float share, u64 sum, bool &whole) {
    const uint32_t bits = __float_as_uint(share), exponent = bits >> 23;
    const u64 digits = exponent > 0 ? (bits & 0x7fffffu) | 0x800000u : bits & 0x7fffffu;
    const int down = 150 - max((int)exponent, 1);  // share = digits / 2^down, 24 <= down <= 149
    const u64 low = digits * sum, high = __umul64hi(digits, sum);
    if (down < 64) {
        whole = (low << (64 - down)) == 0;
        return high << (64 - down) | low >> down;
    }
    const int rest = down - 64;
    const u64 most = rest < 32 ? high >> rest : 0;  // (high is below 2^22)
    whole = low == 0 && (rest < 32 ? most << rest == high : high == 0);
    return most;
}

// What is asked for: the first rank whose running sum exceeds `past`, or, by count, rank number past + 1.
struct Target {
    bool by_count;
    u64 past;
    __device__ __forceinline__ bool within(u64 sum0, uint32_t count0, u64 sum1, uint32_t count1) const {
        return by_count ? count0 <= past && past < count1 : sum0 <= past && past < sum1;
    }
};

// The settings of a row, and what they ask for.
struct Row {
    float temperature, top_p, min_p, u;
    int top_k;
    bool by_p;
    __device__ __forceinline__ Row(const SampleArgs &p, int r)
        : temperature(p.temperatures ? p.temperatures[r] : p.temperature), top_p(p.top_ps ? p.top_ps[r] : p.top_p), min_p(p.min_ps ? p.min_ps[r] : p.min_p),
          u(p.u[r]), top_k(p.top_ks ? p.top_ks[r] : p.top_k), by_p(top_p < 1.0f && top_p > 0.0f) {}
    __device__ __forceinline__ Target k_target() const { return Target{true, (u64)(top_k - 1)}; }
    // the last that top_p keeps of a sum (by_p: 0 < top_p < 1), which the sum that reaches its share ends with, and the drawn one
    __device__ __forceinline__ Target p_target(u64 sum) const {
        bool whole;
        const u64 share = mostof(top_p, sum, whole);
        return Target{false, whole && share > 0 ? share - 1 : share};
    }
    __device__ __forceinline__ Target u_target(u64 sum, u64 first) const {  // first: the weight of the first, which is always kept
        sum = max(top_p <= 0.0f ? first : sum, first);
        bool whole;
        return Target{false, u >= 1.0f ? sum - 1 : u > 0.0f ? mostof(u, sum, whole) : 0ull};
    }
};

// The row's elements, four in a run, SM_AHEAD runs on their way at a time: visit(i, four of them), where those behind the last are NaN.
struct Runs {
    static constexpr int kStep = 4 * SM_THREADS;
    const float *row;
    int n, tid, first;
    float4 x[SM_AHEAD];
    static __device__ __forceinline__ float4 load(const float *row, int n, int i) {
        const int whole = n & ~3;
        return whole > 0 ? load4(row + min(i, max(whole - 4, 0))) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
    __device__ __forceinline__ float4 load(int i) const { return load(row, n, i); }
    // without the first `skip` runs of each thread
    __device__ __forceinline__ Runs(const float *row, int n, int tid, int skip = 0) : row(row), n(n), tid(tid), first(4 * tid + skip * kStep) {
        if (skip * kStep < n)
#pragma unroll
            for (int a = 0; a < SM_AHEAD; ++a) x[a] = load(first + a * kStep);
    }
    template <class F>
    __device__ __forceinline__ void each(F &&visit) {
        const int whole = n & ~3;
#pragma unroll 1
        for (int i = first; i < whole; i += SM_AHEAD * kStep)
#pragma unroll
            for (int a = 0; a < SM_AHEAD; ++a) {
                if (i + a * kStep < whole) visit(i + a * kStep, x[a]);
                x[a] = load(i + (SM_AHEAD + a) * kStep);
            }
        if (whole < n && tid == SM_THREADS - 1) {
            const float nan = __builtin_nanf("");
            visit(whole, make_float4(row[whole], whole + 1 < n ? row[whole + 1] : nan, whole + 2 < n ? row[whole + 2] : nan, nan));
        }
    }
};
__device__ __forceinline__ float max_of_run(const float4 &x) { return fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)); }

__global__ __launch_bounds__(SM_THREADS) void sample_rows_kernel(const SampleArgs p) {
    __shared__ __align__(16) Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x, n = p.n;
    const float *logits = p.logits + (size_t)r * n;
    const Row row(p, r);
    const double temperature = (double)row.temperature > 1e-8 ? fmin((double)row.temperature, 1e39) : 1e-8;
    auto all_max = [&](float v) {  // of the workgroup
        v = wave_max(v);
        __syncthreads();
        if (lane == 0) s.wave_top[wave] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SM_WAVES; ++w) v = fmaxf(v, s.wave_top[w]);
        return v;
    };
    float top = -INFINITY;
    bool infinite = false;  // of a largest logit of infinity only its equals count: they are zeros, the others infinitely less
    auto value = [&](float x) { return !infinite ? x : x == INFINITY ? 0.0f : -INFINITY; };
    Scale scale;
    bool listed = false;  // the list is a first part of the ranking by itself (top_k), or bins of it
    if (tid == 0) s.fill = 0;
    if (tid < SM_LIST) s.place[tid] = 0;

    // ---- the list of a small top_k ----
    if (row.top_k > 0 && row.top_k <= SM_TOP_K && row.top_k < n) {
        // the row's first elements stay in registers for the second look at them
        constexpr int kHeld = 12;
        float4 held[kHeld];
#pragma unroll
        for (int a = 0; a < kHeld; ++a) held[a] = Runs::load(logits, n, 4 * tid + a * Runs::kStep);
#pragma unroll
        for (int a = 0; a < kHeld; ++a)
            if (4 * tid + a * Runs::kStep < (n & ~3)) top = fmaxf(top, max_of_run(held[a]));  // (no element counts for two threads)
        Runs(logits, n, tid, kHeld).each([&](int, const float4 &x) { top = fmaxf(top, max_of_run(x)); });
        s.top[tid] = order_key(top);
        top = all_max(top);
        if (wave == 0) {  // the upper 20 bits of the top_k-th largest maximum, from the first bit on that not all share
            uint32_t mine[SM_WAVES], most = 0u, least = 0xffffffffu;
#pragma unroll
            for (int i = 0; i < SM_WAVES; ++i) {
                mine[i] = s.top[64 * i + lane];
                most = max(most, mine[i]);
                least = min(least, mine[i]);
            }
            most = wave_minmax_u32<true>(most);
            least = wave_minmax_u32<false>(least);
            const int bits = 31 - __builtin_clz((most ^ least) | 1u);
            uint32_t b = bits >= 31 ? 0u : most & ~((2u << bits) - 1u);
#pragma unroll 1
            for (int bit = bits; bit >= 12; --bit) {
                const uint32_t higher = b | (1u << bit);
                int c = 0;
#pragma unroll
                for (int i = 0; i < SM_WAVES; ++i) c += __popcll(__ballot(mine[i] >= higher));
                if (c >= row.top_k) b = higher;
                if (c >= row.top_k && c <= row.top_k + 24) break;  // (some more than needed do no harm)
            }
            if (lane == 0) s.hit[0] = (int)(b & 0xfffff000u);
        }
        __syncthreads();
        const uint32_t bound = (uint32_t)s.hit[0];
        const float floor = key_value(bound);  // (a key between two numbers', or below all of them: NaN, which nothing is below)
        auto list = [&](int i, const float4 &x) {
            if (max_of_run(x) < floor) return;
            const float of[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (order_key(of[e]) >= bound && of[e] > -INFINITY) {
                    const int at = atomicAdd(&s.fill, 1);
                    if (at < SM_LIST) s.list[at] = 1ull << kKeyBits | composite(of[e], i + e);
                }
        };
        Runs more(logits, n, tid, kHeld);
#pragma unroll
        for (int a = 0; a < kHeld; ++a)
            if (4 * tid + a * Runs::kStep < (n & ~3)) list(4 * tid + a * Runs::kStep, held[a]);
        more.each(list);
        __syncthreads();
        listed = s.fill <= SM_LIST && top > -INFINITY && top < INFINITY;
        if (listed) scale.set(top, temperature, p.bits);
        __syncthreads();
        if (!listed && tid == 0) s.fill = 0;
    }

    // ---- the bins ----
    int q_top = 0;  // the bin of the largest logit; bin number j from there on down is j in what follows
    const bool by_k_bins = row.top_k > 0 && row.top_k < n;
    if (!listed) {
        for (int attempt = 0;; ++attempt) {
            for (int i = tid; i < SM_BINS; i += SM_THREADS) {
                s.sum[i] = 0;
                s.count[i] = 0;
            }
            Runs runs(logits, n, tid);
            float seen = attempt == 0 ? max_of_run(runs.x[0]) : top;  // of the first 4096, and then of all
            if (attempt == 0) seen = all_max(seen);
            infinite = seen == INFINITY;
            scale.set(infinite || seen == -INFINITY ? 0.0 : (double)seen, temperature, p.bits);
            __syncthreads();
            top = -INFINITY;
            runs.each([&](int i, const float4 &run) {
                float x[4] = {run.x, run.y, run.z, run.w};
                top = fmaxf(top, max_of_run(run));
                if (__builtin_expect(infinite, 0)) {
                    asm volatile("");  // (a branch, not four selections a run)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = value(x[e]);
                }
                uint32_t id[4];
                u64 weight[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int q = scale.bin(x[e], weight[e]);
                    id[e] = (uint32_t)(scale.counts(x[e]) ? q : Scale::kNone);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (id[e] != (uint32_t)Scale::kNone) {
                        atomicAdd(&s.sum[id[e] & (SM_BINS - 1)], weight[e]);
                        if (by_k_bins) atomicAdd(&s.count[id[e] & (SM_BINS - 1)], 1u);
                    }
                auto two = [&](uint32_t a, uint32_t b) { return (a << kIdShift & 0xffffu) | b << (16 + kIdShift); };
                if (i < SM_IDS) *reinterpret_cast<uint2 *>(&s.id[i]) = make_uint2(two(id[0], id[1]), two(id[2], id[3]));
            });
            top = all_max(top);
            if (top == -INFINITY) {  // nothing to draw from
                if (tid == 0) p.tokens[r] = -1;
                return;
            }
            // (the bins are right, unless the largest is beyond them or has infinite company)
            if (seen > -INFINITY && infinite == (top == INFINITY) && (infinite || top <= scale.high)) break;
        }
        if (infinite) top = 0.0f;
        q_top = scale.bin(top);
        // running sums, in units of the largest logit's bin, from there on down
        u64 w[2];
        uint32_t c[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = 2 * tid + e;
            w[e] = in_units(s.sum[(q_top - j) & (SM_BINS - 1)], units(j)) + (e ? w[0] : 0);
            c[e] = s.count[(q_top - j) & (SM_BINS - 1)] + (e ? c[0] : 0);
        }
        u64 before = sum_up_to(w[1]);
        uint32_t count_before = (uint32_t)sum_up_to(c[1]);
        if (lane == 63) {
            s.wave_sum[wave] = before;
            s.wave_count[wave] = count_before;
        }
        __syncthreads();
        before -= w[1];
        count_before -= c[1];
#pragma unroll
        for (int v = 0; v < SM_WAVES - 1; ++v) {
            before += v < wave ? s.wave_sum[v] : 0;
            count_before += v < wave ? s.wave_count[v] : 0;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            s.sum[2 * tid + e] = before + w[e];
            s.count[2 * tid + e] = count_before + c[e];
        }
        __syncthreads();
    } else {
        q_top = scale.bin(top);
    }
    const u64 first_weight = scale.weight(top);
    auto sum_before = [&](int j) { return !listed && j > 0 ? s.sum[j - 1] : 0; };
    auto count_before = [&](int j) { return !listed && j > 0 ? s.count[j - 1] : 0; };
    // min_p keeps what has at least that weight; in bins m_first .. m_last it is decided
    const bool by_m = row.min_p > 0.0f;
    auto min_p_keeps = [&](float x) { return exp2_wide(fmax(((double)x - top) * (1.4426950408889634 / temperature), -1000.0)) >= (double)row.min_p; };
    // bins of the running sums where two targets lie (s.hit)
    auto find = [&](const Target &a, const Target &b) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = 2 * tid + e;
            if (a.within(sum_before(j), count_before(j), s.sum[j], s.count[j])) s.hit[0] = j;
            if (b.within(sum_before(j), count_before(j), s.sum[j], s.count[j])) s.hit[1] = j;
        }
        __syncthreads();
    };
    const uint32_t candidates = listed ? (uint32_t)s.fill : s.count[SM_BINS - 1];
    const bool by_k = by_k_bins && (uint32_t)row.top_k < candidates;
    int m_first = 0, m_last = 0;
    if (!listed) {
        u64 least = s.sum[SM_BINS - 1], most = least;  // between which what is kept so far adds up to
        int ranges = 0;
        auto range = [&](int from, int to) {
            least = min(least, sum_before(from));
            most = min(most, s.sum[to]);
            if (tid == 0) s.from[ranges] = from, s.to[ranges] = to;
            ++ranges;
            __syncthreads();
        };
        if (by_k) {
            find(row.k_target(), row.k_target());
            range(s.hit[0], s.hit[1]);
        }
        if (row.by_p) {
            find(row.p_target(least), row.p_target(most));
            range(s.hit[0], s.hit[1]);
        }
        if (by_m) {  // (32 times the fp32 logarithm is off by less than 1e-2)
            const double t = ((double)top - scale.origin) * scale.per + SM_OCTAVE * (double)__log2f(fminf(row.min_p, 1.0f));
            auto at = [&](double bin) { return max(q_top - (int)__builtin_rint(fmax(bin, -48.0 * SM_OCTAVE)), 0); };
            m_first = at(t + 1e-2);
            m_last = at(t - 1e-2);
            range(m_first, m_last);
        }
        find(row.u_target(least, first_weight), row.u_target(most, first_weight));
        range(s.hit[0], s.hit[1]);
        // what is in those bins
        // (two elements' bins at a time: how far above a range's last bin a bin lies, less the range's length, is 0 within it)
        u16x2 last[4], length[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int of = min(q, ranges - 1);
            last[q] = (u16x2)(uint16_t)((uint32_t)(q_top - s.to[of]) << kIdShift);
            length[q] = (u16x2)(uint16_t)((s.to[of] - s.from[of]) << kIdShift);
        }
        auto outside = [&](uint32_t two) {
            const u16x2 ids = __builtin_bit_cast(u16x2, two);
            auto of = [&](int q) { return __builtin_elementwise_sub_sat((u16x2)(ids - last[q]), length[q]); };
            u16x2 o = of(0);
            if (ranges > 1) o = __builtin_elementwise_min(o, of(1));
            if (ranges > 2) o = __builtin_elementwise_min(__builtin_elementwise_min(o, of(2)), of(3));
            return o;
        };
        auto put = [&](int i) {
            if (i >= n || *(volatile int *)&s.fill > SM_LIST) return;  // (no more of them when they do not fit anyway)
            const int at = atomicAdd(&s.fill, 1);
            if (at < SM_LIST) s.ranked[at] = (u64)i;
        };
#pragma unroll 1
        for (int i = 8 * tid; i < min(n, SM_IDS); i += 8 * SM_THREADS) {
            const uint4 ids = *reinterpret_cast<const uint4 *>(&s.id[i]);
            const uint32_t of[4] = {ids.x, ids.y, ids.z, ids.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u16x2 o = outside(of[e]);
                if (o.x == 0) put(i + 2 * e);
                if (o.y == 0) put(i + 2 * e + 1);
            }
        }
#pragma unroll 1
        for (int i = SM_IDS + tid; i < n; i += SM_THREADS) {
            const float x = value(logits[i]);
            if (scale.counts(x) && outside((uint32_t)scale.bin(x) << kIdShift & 0xffffu).x == 0) put(i);
        }
        __syncthreads();
        if (tid < min(s.fill, SM_LIST)) {  // their values, all on their way at once
            const int i = (int)s.ranked[tid];
            const float x = value(logits[i]);
            s.list[tid] = (u64)(SM_BINS - 2 - (q_top - scale.bin(x))) << kKeyBits | composite(x, i);  // the bins' order is that of the list too
        }
        __syncthreads();
    }

    // ---- the list in order ----
    auto in_order = [&](int count) {  // list -> ranked
        // the place of an element is the number of elements before it, which `helpers` waves count a part of each
        const int groups = max((count + 63) >> 6, 1), helpers = SM_WAVES / groups, helper = __builtin_amdgcn_readfirstlane(wave / groups), which = tid - 64 * groups * helper;
        if (helper < helpers && which < count) {
            // (as the bits of positive 64-bit floats, whose order is the same: one instruction)
            const double *list = reinterpret_cast<const double *>(s.list), c = list[which];
            int before = 0;
            const int part = (count + helpers - 1) / helpers, last = min((helper + 1) * part, count);
#pragma unroll 4
            for (int o = helper * part; o < last; ++o) before += list[o] > c ? 1 : 0;
            if (before) atomicAdd(&s.place[which], before);
        }
        __syncthreads();
        if (tid < count) s.ranked[s.place[tid]] = s.list[tid];
        __syncthreads();
    };
    auto scanned = [&](u64 w) {  // the sum over the threads up to this one
        w = sum_up_to(w);
        if (lane == 63) s.wave_sum[wave] = w;
        __syncthreads();
        for (int v = 0; v < wave; ++v) w += s.wave_sum[v];
        return w;
    };
    const int in_list = min(s.fill, SM_LIST);
    const bool fits = s.fill <= SM_LIST;
    u64 mine = 0, my_before = 0, my_run = 0;  // of the list's rank tid: the running sums without it and with it
    uint32_t my_rank = 0;
    float my_x = 0.0f;
    if (fits) {
        in_order(in_list);
        u64 weight = 0;
        int j = 0;
        if (tid < in_list) {
            mine = s.ranked[tid];
            my_x = value_of(mine);
            if (scale.counts(my_x)) {
                j = q_top - scale.bin(my_x, weight);
                if (listed) weight = in_units(weight, units(j));  // one by one; otherwise by bins
            }
        }
        const u64 w = scanned(weight);
        s.list[tid] = w;
        __syncthreads();
        if (tid < in_list) {
            if (listed) {
                my_run = w;
                my_before = w - weight;
                my_rank = (uint32_t)tid;
            } else {
                int begin = tid;  // of its bin: the first with the same upper bits
                for (int step = SM_LIST / 2; step > 0; step >>= 1)
                    if (begin - step >= 0 && s.ranked[begin - step] >> kKeyBits == mine >> kKeyBits) begin -= step;
                const double by = units(j);
                const u64 in_bin = w - (begin > 0 ? s.list[begin - 1] : 0);
                my_run = sum_before(j) + in_units(in_bin, by);
                my_before = sum_before(j) + in_units(in_bin - weight, by);
                my_rank = count_before(j) + (uint32_t)(tid - begin);
            }
        }
    }

    // What is in bins first .. last, read from the row again: visit(index, value, bin)
    auto for_bins = [&](int tid, int first, int last, auto &&visit) {
        const int whole = n & ~3;
        float4 next = Runs::load(logits, n, 4 * tid);
#pragma unroll 1
        for (int i = 4 * tid; i < n; i += Runs::kStep) {
            float4 run = next;
            next = Runs::load(logits, n, i + Runs::kStep);
            if (i >= whole) {
                const float nan = __builtin_nanf("");
                run = make_float4(logits[i], i + 1 < n ? logits[i + 1] : nan, i + 2 < n ? logits[i + 2] : nan, nan);
            }
            const float of[4] = {run.x, run.y, run.z, run.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = value(of[e]);
                if (!scale.counts(x)) continue;
                const int j = q_top - scale.bin(x);
                if (j >= first && j <= last) visit(i + e, x, j);
            }
        }
    };

    // ---- top_k, top_p of its sum, min_p, the draw ----
    u64 kept = listed ? s.list[max(in_list - 1, 0)] : s.sum[SM_BINS - 1];
#pragma unroll 1
    for (int stage = 0; stage < 4; ++stage) {
        if (!(stage == 0 ? by_k : stage == 1 ? row.by_p : stage == 2 ? by_m : true)) continue;  // uniform
        __syncthreads();  // the last answer has been read
        if (stage == 2) {
            if (tid == 0) s.kept_of_min_p = sum_before(m_first);
            __syncthreads();
            if (fits) {
                if (tid < in_list && min_p_keeps(my_x)) atomicMax(&s.kept_of_min_p, my_run);
            } else {
                // the weights that are kept in each of these bins (two at most)
                if (tid < SM_PIECES) s.list[tid] = 0;
                __syncthreads();
                int me = tid;
                asm volatile("" : "+v"(me));  // (what follows from it is worked out here, and takes no registers all along)
                for_bins(me, m_first, m_last, [&](int, float x, int j) {
                    if (min_p_keeps(x)) atomicAdd(&s.list[min(j - m_first, SM_PIECES - 1)], scale.weight(x));
                });
                __syncthreads();
                if (tid == 0)
                    for (int j = m_first; j <= min(m_last, m_first + SM_PIECES - 1); ++j)
                        if (s.list[j - m_first] > 0) s.kept_of_min_p = sum_before(j) + in_units(s.list[j - m_first], units(j));
            }
            __syncthreads();
            kept = min(kept, s.kept_of_min_p);
            continue;
        }
        const Target to = stage == 0 ? row.k_target() : stage == 1 ? row.p_target(kept) : row.u_target(kept, first_weight);
        if (fits) {
            if (tid < in_list && to.within(my_before, my_rank, my_run, my_rank + 1)) {
                s.answer_index = (uint32_t)index_of(mine);
                s.answer_sum = my_run;
            }
        } else {
            find(to, to);
            const int j = s.hit[0];
            const double by = units(j);
            const u64 base = sum_before(j);
            const uint32_t rank0 = count_before(j);
            // A piece of the bin: composites from `low` to `high`; before it in the bin lie sum0 and count0.  It is cut by the first nine bits in which its own differ.
            int me = tid;
            asm volatile("" : "+v"(me));
            u64 low = 0, high = ~0ull, sum0 = 0;
            uint32_t count0 = 0;
            int size, shift;
            auto for_piece = [&](auto &&visit) {
                for_bins(me, j, j, [&](int i, float x, int) {
                    const u64 c = composite(x, i);
                    if (c >= low && c <= high) visit(c, x);
                });
            };
            do {
                __syncthreads();
                if (tid < SM_PIECES) {
                    s.list[tid] = 0;
                    s.place[tid] = 0;
                }
                if (tid == 0) {
                    s.least = ~0ull;
                    s.most = 0;
                }
                __syncthreads();
                u64 least = ~0ull, most = 0;
                for_piece([&](u64 c, float) {
                    least = min(least, c);
                    most = max(most, c);
                });
                if (least <= most) {
                    atomicMin(&s.least, least);
                    atomicMax(&s.most, most);
                }
                __syncthreads();
                least = s.least;
                const int bit = 63 - __builtin_clzll((least ^ s.most) | 1ull);
                shift = max(bit - 8, 0);
                const u64 mask = (2ull << (bit - shift)) - 1, common = least >> shift & ~mask;
                for_piece([&](u64 c, float x) {
                    const int d = SM_PIECES - 1 - (int)(c >> shift & mask);
                    atomicAdd(&s.list[d], scale.weight(x));
                    atomicAdd(&s.place[d], 1);
                });
                __syncthreads();
                const u64 mine = tid < SM_PIECES ? s.list[tid] : 0;
                const uint32_t count = tid < SM_PIECES ? (uint32_t)s.place[tid] : 0;
                const u64 upto = sum0 + scanned(mine);
                __syncthreads();
                const uint32_t counted = count0 + (uint32_t)scanned(count);
                if (count > 0 && to.within(base + in_units(upto - mine, by), rank0 + counted - count, base + in_units(upto, by), rank0 + counted)) {
                    s.piece = tid;
                    s.piece_sum = upto - mine;
                    s.piece_count = counted - count;
                }
                __syncthreads();
                size = s.place[s.piece];
                sum0 = s.piece_sum;
                count0 = s.piece_count;
                low = (common | (u64)(SM_PIECES - 1 - s.piece)) << shift;
                high = low + ((1ull << shift) - 1);
            } while (size > SM_PIECE && shift > 0);
            __syncthreads();
            if (tid == 0) s.fill = 0;
            s.place[tid] = 0;
            __syncthreads();
            for_piece([&](u64 c, float) { s.list[min(atomicAdd(&s.fill, 1), SM_LIST - 1)] = 1ull << kKeyBits | c; });
            __syncthreads();
            in_order(size);
            const u64 c = tid < size ? s.ranked[tid] : 0, weight = tid < size ? scale.weight(value_of(c)) : 0, with = sum0 + scanned(weight);
            if (tid < size && to.within(base + in_units(with - weight, by), rank0 + count0 + (uint32_t)tid, base + in_units(with, by), rank0 + count0 + (uint32_t)tid + 1)) {
                s.answer_index = (uint32_t)index_of(c);
                s.answer_sum = base + in_units(with, by);
            }
        }
        __syncthreads();
        kept = min(kept, s.answer_sum);
    }
    if (tid == 0) p.tokens[r] = (int)s.answer_index;
}

}  // namespace

AGPU_EXPORT int32_t agpu_sample(agpu_ctx *ctx, const float *logits, const float *u, int32_t *tokens_out, int32_t rows, int32_t n, float temperature,
                                int32_t top_k, float top_p, float min_p, const float *temperatures, const int32_t *top_ks, const float *top_ps,
                                const float *min_ps) {
    AGPU_REQUIRE_CTX(ctx);
    if (rows < 0 || n <= 0) return agpu_fail(ctx, AGPU_ERR_SHAPE_MISMATCH, "sample: bad dims rows=%d n=%d", rows, n);
    if (n > 1 << kIndexBits) return agpu_fail(ctx, AGPU_ERR_UNSUPPORTED, "sample: n = %d exceeds %d", n, 1 << kIndexBits);
    if (rows >= 1 << 22) return agpu_fail(ctx, AGPU_ERR_UNSUPPORTED, "sample: %d rows", rows);
    if (rows == 0) return AGPU_OK;
    if (!logits || !u || !tokens_out) return agpu_fail(ctx, AGPU_ERR_NULL_POINTER, "sample: null pointer");
    agpu_on_device here(ctx);
    if (here.rc != AGPU_OK) return here.rc;
    const int bits = std::min(61 - (n > 1 ? 32 - __builtin_clz(n - 1) : 0), 50);
    const SampleArgs p = {logits, u, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p, top_k, tokens_out, n, bits};
    hipLaunchKernelGGL(sample_rows_kernel, dim3(rows), dim3(SM_THREADS), 0, ctx->stream, p);
    return AGPU_LAUNCH_CHECK(ctx, "sample_rows_kernel");
}
