// The draw of the next tokens from rows of logits: temperature, top-k, top-p and min-p, and one given number of [0, 1) a row.
//   w_i = exp((x_i - max) / T); candidates ranked by x, the largest first, the lower index first among equals.
// Each filter keeps a first part of the ranking (the k first; those before which less than p of the k's sum lies; w >= min_p), so that what is kept is the
// shortest of the three parts, and all that the draw needs of it is its sum Z: the token is the first rank whose running sum exceeds u Z.
//
// Sums decide, next to borders, which token comes out, and there are tens of thousands of terms: weights are whole numbers, w 2^46 at
// 50257 logits, from an exponential in 64-bit floats (off by 4e-14 of itself), and their sums are exact in any order.  (With fp32 exponentials a row of
// 50257 logits would go wrong about once in a thousand draws.)
//
// Three launches, of a few workgroups a row each, which take a part of it; what they find they add to the row's state in memory, and the last one of a
// row to finish draws the conclusion.
//   sample_top_kernel    the parts' maxima
//   sample_bins_kernel   sums (and counts, where top_k asks for them) of the weights in 2048 bins of log2 w.  From their running sums follows in which bins the
//                        filters' borders lie, between which sums Z then is, and in which bins the drawn rank can be: up to three ranges of bins
//   sample_draw_kernel   what is in those bins, a few hundred elements, is gathered, put in order by counting, and searched
// When the bins hold too many (thousands of equal logits, a large temperature), the last workgroup looks for each border by itself, in bins cut into
// 2048 by the bits of (value, index), which are never the same twice, until a piece fits the list.
#include "agpu_internal.h"
#include "sampling.h"

#include <algorithm>

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 512, SM_WAVES = SM_THREADS / 64;
constexpr int SM_BINS = 2048, SM_LIST = 512, SM_MAX_PARTS = 32, SM_PARTS = 256;  // SM_PARTS: workgroups of a launch, about
constexpr int SM_AHEAD = 4;  // runs of four elements that a thread has on their way at a time
constexpr int kIndexBits = 20;  // n <= 2^20

struct SampleArgs {
    const float *logits, *u;
    const float *temperatures, *top_ps, *min_ps;
    const int *top_ks;
    float temperature, top_p, min_p;
    int top_k;
    int *tokens;
    int n, bits;  // bits of a weight of one: sums of n weights stay below 2^62, and of one below 2^51
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

struct Scale {
    double top, per, least;  // the largest logit; log2(e) / T; log2 of what is no weight any more, less than half a unit
    float bins_per_octave;   // so that the last bin is not passed
    int bits;
    __device__ __forceinline__ Scale(float top_, float temperature, int bits_)
        : top(top_), per(1.4426950408889634 / ((double)temperature > 1e-8 ? (double)temperature : 1e-8)), least(-(bits_ + 1)),
          bins_per_octave((SM_BINS - 0.125f) / (bits_ + 1)), bits(bits_) {}
    __device__ __forceinline__ double log2_of(float x) const { return ((double)x - top) * per; }
    __device__ __forceinline__ bool counts(double t) const { return t > least; }  // (NaN does not)
    // To the nearest whole number.  1.5 2^52 more leaves the nearest one of t, and 2^52 more that of the weight, in the low bits.
    __device__ __forceinline__ u64 weight(double t) const {
        const double shifted = t + 0x1.8p52;
        const u64 y = __builtin_bit_cast(u64, exp2_part(t - (shifted - 0x1.8p52)));
        const u64 exponent = (u64)((uint32_t)__builtin_bit_cast(u64, shifted) + (uint32_t)bits) << 52;
        return __builtin_bit_cast(u64, __builtin_bit_cast(double, y + exponent) + 0x1p52) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ int bin(double t) const { return (int)((float)-t * bins_per_octave); }
};

__device__ __forceinline__ u64 composite(float x, int i) { return (u64)order_key(x) << kIndexBits | (u64)((1 << kIndexBits) - 1 - i); }
__device__ __forceinline__ float value_of(u64 c) { return key_value((uint32_t)(c >> kIndexBits)); }
__device__ __forceinline__ int index_of(u64 c) { return (1 << kIndexBits) - 1 - (int)(c & ((1 << kIndexBits) - 1)); }

// What the launches leave for one another of a row.
struct RowState {
    u64 sum[SM_BINS], min_p_sum;  // of the bins; of the weights from min_p on
    uint32_t count[SM_BINS];
    float top[SM_MAX_PARTS];
    int ranges, first[3], last[3];  // bins where borders and the drawn rank can be
    u64 more_sum[3];                // the running sum and count before a range less what the list holds before it
    uint32_t more_count[3];
    u64 all;                        // sum and number of all candidates
    uint32_t candidates;
    uint32_t fill;
    u64 list[SM_LIST];
};
struct Parts {
    int n, each, row0;  // parts of a row and elements of each (a multiple of four); the first row of the launch
    RowState *rows;
    unsigned int *tickets;
    int strict;
};

struct Bins {
    u64 sum[SM_BINS], wave_sum[SM_WAVES], hit_sum[2];
    uint32_t count[SM_BINS], wave_count[SM_WAVES], hit_count[2];
    int hit[2];
};

// Sums and counts become running ones from bin 0 on.  Whole workgroup; barriers before and after.
__device__ __forceinline__ void running(Bins &s, int tid, int lane, int wave) {
    constexpr int EACH = SM_BINS / SM_THREADS;
    __syncthreads();
    u64 w[EACH];
    uint32_t c[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        w[e] = s.sum[EACH * tid + e] + (e ? w[e - 1] : 0);
        c[e] = s.count[EACH * tid + e] + (e ? c[e - 1] : 0);
    }
    u64 before = w[EACH - 1];
    uint32_t count_before = c[EACH - 1];
#pragma unroll
    for (int by = 1; by < 64; by <<= 1) {
        const u64 o = __shfl_up(before, by, kWave);
        const uint32_t oc = __shfl_up(count_before, by, kWave);
        if (lane >= by) {
            before += o;
            count_before += oc;
        }
    }
    if (lane == 63) {
        s.wave_sum[wave] = before;
        s.wave_count[wave] = count_before;
    }
    __syncthreads();
    before -= w[EACH - 1];
    count_before -= c[EACH - 1];
    for (int v = 0; v < wave; ++v) {
        before += s.wave_sum[v];
        count_before += s.wave_count[v];
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        s.sum[EACH * tid + e] = before + w[e];
        s.count[EACH * tid + e] = count_before + c[e];
    }
    __syncthreads();
}

// What is asked for: the first rank whose running sum exceeds `past`, or, by count, rank number past + 1.
struct Target {
    bool by_count;
    u64 past;
    __device__ __forceinline__ bool within(u64 sum0, uint32_t count0, u64 sum1, uint32_t count1) const {
        return by_count ? count0 <= past && past < count1 : sum0 <= past && past < sum1;
    }
};

// The bins of running sums (which begin at sum0 and count0) where two targets lie: s.hit, and the sum and count before them.  A barrier at the end.
__device__ __forceinline__ void find(Bins &s, u64 sum0, uint32_t count0, const Target &a, const Target &b, int tid) {
#pragma unroll 1
    for (int x = tid; x < SM_BINS; x += SM_THREADS) {
        const u64 s0 = sum0 + (x ? s.sum[x - 1] : 0), s1 = sum0 + s.sum[x];
        const uint32_t c0 = count0 + (x ? s.count[x - 1] : 0), c1 = count0 + s.count[x];
        auto look = [&](int i, const Target &to) {
            if (!to.within(s0, c0, s1, c1)) return;
            s.hit[i] = x;
            s.hit_sum[i] = s0;
            s.hit_count[i] = c0;
        };
        look(0, a);
        look(1, b);
    }
    __syncthreads();
}

// The settings of a row, and what they ask for.
struct Row {
    float temperature, top_p, min_p, u;
    int top_k;
    u64 one;
    bool by_p;
    __device__ __forceinline__ Row(const SampleArgs &p, int r)
        : temperature(p.temperatures ? p.temperatures[r] : p.temperature), top_p(p.top_ps ? p.top_ps[r] : p.top_p), min_p(p.min_ps ? p.min_ps[r] : p.min_p),
          u(p.u[r]), top_k(p.top_ks ? p.top_ks[r] : p.top_k), one(1ull << p.bits), by_p(top_p < 1.0f && top_p > 0.0f) {}
    // Stages 0: the last of top_k, 1: the last that top_p keeps of the sum `kept`, 2: the drawn one of it
    __device__ __forceinline__ bool asked(int stage, uint32_t candidates) const {
        return stage == 0 ? top_k > 0 && (uint32_t)top_k < candidates : stage == 1 ? by_p : true;
    }
    __device__ __forceinline__ Target target(int stage, u64 kept, u64 min_p_sum) const {
        if (stage == 0) return Target{true, (u64)(top_k - 1)};
        if (stage == 1) {
            const double share = __builtin_ceil((double)top_p * (double)kept) - 1;
            return Target{false, share > 0.0 && kept > 0 ? min((u64)share, kept - 1) : 0ull};
        }
        if (top_p <= 0.0f) kept = one;
        if (min_p > 0.0f) kept = min(kept, min_p_sum);
        kept = max(kept, one);  // the first is always kept
        const double at = (double)u * (double)kept;
        return Target{false, at > 0.0 ? min((u64)at, kept - 1) : 0ull};
    }
};

// The elements lo .. hi - 1 of a row, four in a run, SM_AHEAD runs on their way at a time: visit(i, four of them), where those behind the last are NaN.
// (Few copies of visit: code comes cold from memory at every launch.)
template <int THREADS, class F>
__device__ __forceinline__ void for_runs(const float *row, int lo, int hi, int tid, F &&visit) {
    const int whole = hi - (hi - lo) % 4, step = 4 * THREADS;
    if (lo >= hi) return;
    float4 x[SM_AHEAD];
    const int back = max(whole - 4, lo);
    auto load = [&](int i) { return whole > lo ? load4(row + min(i, back)) : make_float4(0.f, 0.f, 0.f, 0.f); };
    int i = lo + 4 * tid;
#pragma unroll
    for (int a = 0; a < SM_AHEAD; ++a) x[a] = load(i + a * step);
#pragma unroll 1
    for (; i < whole; i += SM_AHEAD * step)
#pragma unroll
        for (int a = 0; a < SM_AHEAD; ++a) {
            if (i + a * step < whole) visit(i + a * step, x[a]);
            x[a] = load(i + (SM_AHEAD + a) * step);
        }
    if (whole < hi && tid == 0) {
        const float nan = __builtin_nanf("");
        visit(whole, make_float4(row[whole], whole + 1 < hi ? row[whole + 1] : nan, whole + 2 < hi ? row[whole + 2] : nan, nan));
    }
}
// Of a largest logit of infinity only its equals count: they are zeros, the others infinitely less.
__device__ __forceinline__ void values(const float4 &run, bool infinite, float (&x)[4]) {
    x[0] = run.x; x[1] = run.y; x[2] = run.z; x[3] = run.w;
    if (__builtin_expect(infinite, 0)) {
        asm volatile("");  // (a branch, not four selections a run)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = x[e] == INFINITY ? 0.0f : -INFINITY;
    }
}

// The last workgroup of a row to arrive (whole workgroup; `ticket` in LDS).
__device__ __forceinline__ bool last_of_row(const Parts &parts, int r, uint32_t &ticket, int tid) {
    if (parts.n == 1) return true;
    partials_published(parts.strict);
    __syncthreads();
    if (tid == 0) {
        ticket = take_ticket(&parts.tickets[r], parts.strict);
        if (ticket == (unsigned)(parts.n - 1)) __hip_atomic_store(&parts.tickets[r], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (ticket != (unsigned)(parts.n - 1)) return false;
    if (parts.strict) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    return true;
}

// grid (parts, rows) here and below: the maximum of a part, and zeros for its share of the bins
__global__ __launch_bounds__(SM_THREADS) void sample_top_kernel(const SampleArgs p, const Parts parts) {
    __shared__ float s_top[SM_WAVES];
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    RowState &state = parts.rows[r];
    for (int i = part * SM_THREADS + tid; i < SM_BINS; i += parts.n * SM_THREADS) {
        state.sum[i] = 0;
        state.count[i] = 0;
    }
    if (part == 0 && tid == 0) {
        state.min_p_sum = 0;
        state.fill = 0;
    }
    float top = -INFINITY;
    const int lo = min(part * parts.each, p.n);
    for_runs<SM_THREADS>(p.logits + (size_t)(parts.row0 + r) * p.n, lo, min(lo + parts.each, p.n), tid,
                         [&](int, const float4 &x) { top = fmaxf(top, fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w))); });
    top = wave_max(top);
    if ((tid & 63) == 0) s_top[tid >> 6] = top;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < SM_WAVES; ++w) top = fmaxf(top, s_top[w]);
        state.top[part] = top;
    }
}

__global__ __launch_bounds__(SM_THREADS) void sample_bins_kernel(const SampleArgs p, const Parts parts) {
    __shared__ Bins s;
    __shared__ u64 s_min_p_sum;
    __shared__ uint32_t s_ticket;
    __shared__ int s_from[3], s_to[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.y;
    const float *logits = p.logits + (size_t)(parts.row0 + r) * p.n;
    RowState &state = parts.rows[r];
    const Row row(p, parts.row0 + r);
    const float top = wave_max(lane < parts.n ? state.top[lane] : -INFINITY);
    if (top == -INFINITY) return;  // nothing to draw from (the whole row)
    const bool infinite = top == INFINITY, counts = row.top_k > 0;
    const Scale scale(infinite ? 0.0f : top, row.temperature, p.bits);
    for (int i = tid; i < SM_BINS; i += SM_THREADS) {
        s.sum[i] = 0;
        s.count[i] = 0;
    }
    if (tid == 0) s_min_p_sum = 0;
    __syncthreads();
    const u64 least = row.min_p > 0.0f ? (u64)__builtin_ceil(fmin((double)row.min_p, 2.0) * (double)row.one) : ~0ull;
    u64 above = 0;  // sum of the weights from min_p on
    const int lo = min((int)blockIdx.x * parts.each, p.n);
    for_runs<SM_THREADS>(logits, lo, min(lo + parts.each, p.n), tid, [&](int, const float4 &run) {
        float x[4];
        values(run, infinite, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double t = scale.log2_of(x[e]);
            if (!scale.counts(t)) continue;
            const u64 w = scale.weight(t);
            const int b = scale.bin(t);
            atomicAdd(&s.sum[b], w);
            if (counts) atomicAdd(&s.count[b], 1u);
            above += w >= least ? w : 0;
        }
    });
    if (row.min_p > 0.0f) {
#pragma unroll
        for (int by = 32; by > 0; by >>= 1) above += __shfl_xor(above, by, kWave);
        if (lane == 0) atomicAdd(&s_min_p_sum, above);
    }
    __syncthreads();
    for (int i = tid; i < SM_BINS; i += SM_THREADS)
        if (s.sum[i] != 0 || s.count[i] != 0) {
            __hip_atomic_fetch_add(&state.sum[i], s.sum[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (counts) __hip_atomic_fetch_add(&state.count[i], s.count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    if (tid == 0 && row.min_p > 0.0f) __hip_atomic_fetch_add(&state.min_p_sum, s_min_p_sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!last_of_row(parts, r, s_ticket, tid)) return;
    if (parts.n > 1) {
        for (int i = tid; i < SM_BINS; i += SM_THREADS) {
            s.sum[i] = __hip_atomic_load(&state.sum[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s.count[i] = counts ? __hip_atomic_load(&state.count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
        }
        if (tid == 0) s_min_p_sum = __hip_atomic_load(&state.min_p_sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    running(s, tid, lane, wave);
    auto sum_before = [&](int b) { return b > 0 ? s.sum[b - 1] : 0; };
    u64 least_sum = s.sum[SM_BINS - 1], most_sum = least_sum;  // between which what is kept so far adds up to
    const uint32_t candidates = s.count[SM_BINS - 1];
#pragma unroll 1
    for (int stage = 0; stage < 3; ++stage) {
        if (!row.asked(stage, candidates)) continue;  // uniform
        find(s, 0, 0, row.target(stage, least_sum, s_min_p_sum), row.target(stage, most_sum, s_min_p_sum), tid);
        least_sum = min(least_sum, sum_before(s.hit[0]));
        most_sum = min(most_sum, s.sum[s.hit[1]]);
        if (tid == 0) s_from[stage] = s.hit[0], s_to[stage] = s.hit[1];
        __syncthreads();
    }
    if (tid != 0) return;
    // What is drawn does not come behind the last that top_p keeps, nor that behind the last of top_k: the ranges are in order.  Those that meet are one.
    int n = 0, begin = 0, end = -2;
    u64 sum = 0;
    uint32_t count = 0;
#pragma unroll 1
    for (int stage = 2; stage >= 0; --stage) {
        if (!row.asked(stage, candidates)) continue;
        const int a = max(s_from[stage], 0), b = s_to[stage];
        if (n > 0 && a <= end + 1) {
            end = max(end, b);
            state.last[n - 1] = end;
            continue;
        }
        if (n > 0) {  // the range before is complete
            sum += s.sum[end] - sum_before(begin);
            count += s.count[end] - (begin ? s.count[begin - 1] : 0);
        }
        begin = a;
        state.first[n] = a;
        state.last[n] = end = b;
        state.more_sum[n] = sum_before(a) - sum;
        state.more_count[n] = (a ? s.count[a - 1] : 0) - count;
        ++n;
    }
    state.ranges = n;
    state.all = s.sum[SM_BINS - 1];
    state.candidates = candidates;
}

__global__ __launch_bounds__(SM_THREADS, 4) void sample_draw_kernel(const SampleArgs p, const Parts parts) {
    __shared__ Bins s;  // (for rows whose list does not hold what it should)
    __shared__ u64 s_list[SM_LIST], s_ranked[SM_LIST], s_answer_sum;
    __shared__ int s_place[SM_LIST];
    __shared__ uint32_t s_fill, s_base, s_ticket, s_answer;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.y, n = p.n;
    const float *logits = p.logits + (size_t)(parts.row0 + r) * n;
    int *const token = p.tokens + parts.row0 + r;
    RowState &state = parts.rows[r];
    const Row row(p, parts.row0 + r);
    const float top = wave_max(lane < parts.n ? state.top[lane] : -INFINITY);
    if (top == -INFINITY) {  // the whole row
        if (tid == 0 && blockIdx.x == 0) *token = -1;
        return;
    }
    const bool infinite = top == INFINITY;
    const Scale scale(infinite ? 0.0f : top, row.temperature, p.bits);
    struct Ranges {
        int n, first[3], last[3];
    };
    // visit(i, x, t, bin) of the part's (or the row's) elements in bins first[q] .. last[q] of the ranges q < n
    auto for_bins = [&](const Ranges &of, int lo, int hi, auto &&visit) {
        // What cannot be in them is told apart by its value alone: a hair beyond the bins' ends (t and the ends round by 2^-23 at most).
        float below[3], above[3];
        const double slack = 1e-5, width = 1.0 / scale.bins_per_octave, by = 1.0 / scale.per;
        auto beyond = [](float x, float by) { return fabsf(x) < INFINITY ? x + fabsf(x) * by : x; };
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            below[q] = beyond((float)(scale.top - ((of.last[q] + 1) * width * (1 + slack) + slack) * by), -1e-6f);
            above[q] = of.first[q] == 0 ? INFINITY : beyond((float)(scale.top - (of.first[q] * width * (1 - slack) - slack) * by), 1e-6f);
            if (q >= of.n) below[q] = INFINITY, above[q] = -INFINITY;
        }
        const float lowest = fminf(below[0], fminf(below[1], below[2]));
        for_runs<SM_THREADS>(logits, lo, hi, tid, [&](int i, const float4 &run) {
            float x[4];
            values(run, infinite, x);
            if (!(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= lowest)) return;
            unsigned near = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                near |= ((x[e] >= below[0] && x[e] <= above[0]) || (x[e] >= below[1] && x[e] <= above[1]) || (x[e] >= below[2] && x[e] <= above[2])) ? 1u << e : 0u;
#pragma unroll 1
            for (; near != 0; near &= near - 1) {
                const int e = __builtin_ctz(near);
                const float y = e < 2 ? (e == 0 ? x[0] : x[1]) : e == 2 ? x[2] : x[3];
                const double t = scale.log2_of(y);
                const int b = scale.counts(t) ? scale.bin(t) : SM_BINS;
                if ((b >= of.first[0] && b <= of.last[0]) || (of.n > 1 && b >= of.first[1] && b <= of.last[1]) || (of.n > 2 && b >= of.first[2] && b <= of.last[2]))
                    visit(i + e, y, t);
            }
        });
    };
    if (tid == 0) s_fill = 0;
    if (tid < SM_LIST) s_place[tid] = 0;
    __syncthreads();
    const Ranges of = {state.ranges, {state.first[0], state.first[1], state.first[2]}, {state.last[0], state.last[1], state.last[2]}};
    const int lo = min((int)blockIdx.x * parts.each, n);
    for_bins(of, lo, min(lo + parts.each, n), [&](int i, float x, double) {
        const uint32_t at = atomicAdd(&s_fill, 1u);
        if (at < SM_LIST) s_list[at] = composite(x, i);
    });
    __syncthreads();
    uint32_t listed = s_fill;
    if (parts.n > 1) {
        if (tid == 0) s_base = __hip_atomic_fetch_add(&state.fill, listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        for (uint32_t i = tid; i < listed && s_base + i < SM_LIST; i += SM_THREADS)
            __hip_atomic_store(&state.list[s_base + i], s_list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (!last_of_row(parts, r, s_ticket, tid)) return;
        listed = __hip_atomic_load(&state.fill, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (uint32_t i = tid; i < min(listed, (uint32_t)SM_LIST); i += SM_THREADS) s_list[i] = __hip_atomic_load(&state.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
    }
    const bool fits = listed <= SM_LIST;
    u64 my_run = 0, my_weight = 0, mine = 0;  // of the list's rank tid
    uint32_t my_rank = 0;
    const u64 min_p_sum = __hip_atomic_load(&state.min_p_sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (fits) {
        // the place of an element is the number of elements before it, which `helpers` threads count a part of each
        const int per = listed > 1 ? 1 << (32 - __builtin_clz(listed - 1)) : 1, helpers = SM_THREADS / per, which = tid & (per - 1), helper = tid / per;
        if (which < (int)listed) {
            const u64 c = s_list[which];
            int before = 0;
            for (int o = helper; o < (int)listed; o += helpers) before += s_list[o] > c ? 1 : 0;
            atomicAdd(&s_place[which], before);
        }
        __syncthreads();
        if (tid < (int)listed) s_ranked[s_place[tid]] = s_list[tid];
        __syncthreads();
        int q = 0;
        if (tid < (int)listed) {
            mine = s_ranked[tid];
            const double t = scale.log2_of(value_of(mine));
            const int b = scale.bin(t);
            q = of.n > 2 && b >= of.first[2] ? 2 : of.n > 1 && b >= of.first[1] ? 1 : 0;
            my_weight = scale.weight(t);
        }
        u64 w = my_weight;
#pragma unroll
        for (int by = 1; by < 64; by <<= 1) {
            const u64 o = __shfl_up(w, by, kWave);
            if (lane >= by) w += o;
        }
        if (lane == 63) s.wave_sum[wave] = w;
        __syncthreads();
        for (int v = 0; v < wave; ++v) w += s.wave_sum[v];
        my_run = w + state.more_sum[q];
        my_rank = (uint32_t)tid + state.more_count[q];
    }
    // the bins' running sums again, where the whole row has to be gone through
    auto load_bins = [&]() {
        __syncthreads();
        for (int i = tid; i < SM_BINS; i += SM_THREADS) {
            s.sum[i] = __hip_atomic_load(&state.sum[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s.count[i] = __hip_atomic_load(&state.count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        running(s, tid, lane, wave);
    };
    u64 kept = ~0ull;
    uint32_t candidates = ~0u;
    if (!fits) {
        load_bins();
        kept = s.sum[SM_BINS - 1];
        candidates = s.count[SM_BINS - 1];
        __syncthreads();
    } else {
        kept = state.all;
        candidates = state.candidates;
    }
#pragma unroll 1
    for (int stage = 0; stage < 3; ++stage) {
        if (!row.asked(stage, candidates)) continue;
        const Target to = row.target(stage, kept, min_p_sum);
        if (fits) {
            if (tid < (int)listed && to.within(my_run - my_weight, my_rank, my_run, my_rank + 1)) {
                s_answer = (uint32_t)index_of(mine);
                s_answer_sum = my_run;
            }
            __syncthreads();
            kept = min(kept, s_answer_sum);
            __syncthreads();
            continue;
        }
        load_bins();
        find(s, 0, 0, to, to, tid);
        const int b = s.hit[0];
        u64 prefix = 0, sum0 = s.hit_sum[0];
        uint32_t count0 = s.hit_count[0], in_piece = SM_LIST + 1;  // (counts there are only where top_k asks for them)
        const Ranges bin = {1, {b, 0, 0}, {b, 0, 0}};
        int known = 52;  // the bits of a composite; those from `known` on are the same, `prefix`
        while (in_piece > SM_LIST && known > 0) {
            const int shift = max(known - 11, 0);
            __syncthreads();
            for (int i = tid; i < SM_BINS; i += SM_THREADS) {
                s.sum[i] = 0;
                s.count[i] = 0;
            }
            __syncthreads();
            for_bins(bin, 0, n, [&](int i, float x, double t) {
                const u64 c = composite(x, i);
                if (c >> known != prefix) return;
                const int d = SM_BINS - 1 - (int)((c >> shift) & ((1ull << (known - shift)) - 1));
                atomicAdd(&s.sum[d], scale.weight(t));
                atomicAdd(&s.count[d], 1u);
            });
            running(s, tid, lane, wave);
            find(s, sum0, count0, to, to, tid);
            const int d = s.hit[0];
            in_piece = s.count[d] - (d ? s.count[d - 1] : 0);
            sum0 = s.hit_sum[0];
            count0 = s.hit_count[0];
            prefix = prefix << (known - shift) | (u64)(SM_BINS - 1 - d);
            known = shift;
        }
        if (tid == 0) s_fill = 0;
        __syncthreads();
        for_bins(bin, 0, n, [&](int i, float x, double) {
            const u64 c = composite(x, i);
            if (c >> known == prefix) s_list[min(atomicAdd(&s_fill, 1u), (uint32_t)SM_LIST - 1)] = c;
        });
        __syncthreads();
        if (tid < (int)in_piece) {
            const u64 c = s_list[tid];
            u64 before = sum0;
            uint32_t rank = count0;
            for (int o = 0; o < (int)in_piece; ++o)
                if (s_list[o] > c) {
                    before += scale.weight(scale.log2_of(value_of(s_list[o])));
                    ++rank;
                }
            const u64 run = before + scale.weight(scale.log2_of(value_of(c)));
            if (to.within(before, rank, run, rank + 1)) {
                s_answer = (uint32_t)index_of(c);
                s_answer_sum = run;
            }
        }
        __syncthreads();
        kept = min(kept, s_answer_sum);
        __syncthreads();
    }
    if (tid == 0) *token = (int)s_answer;
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
    const int bits = std::min(62 - (n > 1 ? 32 - __builtin_clz(n - 1) : 0), 50);
    const SampleArgs p = {logits, u, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p, top_k, tokens_out, n, bits};
    // Rows by as many as the scratch holds the states of; parts of 2048 elements at least.
    const int at_once = (int)std::min<size_t>({(size_t)rows, ctx->ws_bytes / 2 / sizeof(RowState), (size_t)ctx->n_counters - 1, 65535});
    const int count = std::max(1, std::min({SM_PARTS / at_once, n / 2048, SM_MAX_PARTS}));
    for (int row0 = 0; row0 < rows; row0 += at_once) {
        const Parts parts = {count, (ceil_div(n, count) + 3) & ~3, row0, reinterpret_cast<RowState *>(ctx->workspace), ctx->counters, ctx->strict_sync};
        const dim3 grid(count, std::min(at_once, rows - row0));
        hipLaunchKernelGGL(sample_top_kernel, grid, dim3(SM_THREADS), 0, ctx->stream, p, parts);
        hipLaunchKernelGGL(sample_bins_kernel, grid, dim3(SM_THREADS), 0, ctx->stream, p, parts);
        hipLaunchKernelGGL(sample_draw_kernel, grid, dim3(SM_THREADS), 0, ctx->stream, p, parts);
    }
    return AGPU_LAUNCH_CHECK(ctx, "sample kernels");
}
