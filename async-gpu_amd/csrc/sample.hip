// The draw of the next tokens from rows of logits: temperature, top-k, top-p and min-p, and one given number of [0, 1) a row.
//   w_i = exp((x_i - max) / T); candidates ranked by x, the largest first, the lower index first among equals.
// Each filter keeps a first part of the ranking (the k first; those before which less than p of the k's sum lies; w >= min_p), so that what is kept is the
// shortest of the three parts, and all that the draw needs of it is its sum Z: the token is the first rank whose running sum exceeds u Z.
//
// Sums decide, next to borders, which token comes out, and there are tens of thousands of terms: weights are whole numbers, w 2^46 at
// 50257 logits, from an exponential in 64-bit floats (off by 4e-14 of itself), and their sums are exact in any order.  (With fp32 exponentials a row of
// 50257 logits would go wrong about once in a thousand draws.)
//
// sample_rows_kernel, a workgroup a row: the maximum; sums and counts of the weights in 2048 bins of log2 w; then up to three times the rank where a running sum
// (or count) passes a target: its bin from the bins' running sums, and within it from the bin's elements, put in order by counting, together with as
// many bins before it as the list has room for, so that the next target, which is smaller, is often answered from the same list.
// A bin with more elements than that is cut into 2048 by the bits of (value, index), which are never the same twice, until a piece fits.
#include "agpu_internal.h"
#include "sampling.h"

#include <algorithm>

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 1024, SM_WAVES = SM_THREADS / 64;
constexpr int SM_BINS = 2048, SM_LIST = 512;
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
    float bins_per_octave;
    int bits;
    __device__ __forceinline__ Scale(float top_, float temperature, int bits_)
        : top(top_), per(1.4426950408889634 / ((double)temperature > 1e-8 ? (double)temperature : 1e-8)), least(-(bits_ + 1)),
          bins_per_octave((float)SM_BINS / (bits_ + 1)), bits(bits_) {}
    __device__ __forceinline__ double log2_of(float x) const { return (double)x == top ? 0.0 : ((double)x - top) * per; }
    __device__ __forceinline__ bool counts(double t) const { return t > least; }  // (NaN does not)
    __device__ __forceinline__ u64 weight(double t) const {  // to the nearest whole number, which 2^52 more leaves in the low bits
        const double k = __builtin_rint(t);
        const double y = __builtin_amdgcn_ldexp(exp2_part(t - k), (int)k + bits) + 0x1p52;
        return __builtin_bit_cast(u64, y) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ int bin(double t) const { return min((int)((float)-t * bins_per_octave), SM_BINS - 1); }
};

__device__ __forceinline__ u64 composite(float x, int i) { return (u64)order_key(x) << kIndexBits | (u64)((1 << kIndexBits) - 1 - i); }
__device__ __forceinline__ float value_of(u64 c) { return key_value((uint32_t)(c >> kIndexBits)); }
__device__ __forceinline__ int index_of(u64 c) { return (1 << kIndexBits) - 1 - (int)(c & ((1 << kIndexBits) - 1)); }

struct Shared {
    u64 sum[SM_BINS], fine_sum[SM_BINS];
    uint32_t count[SM_BINS], fine_count[SM_BINS];
    u64 list[SM_LIST], ranked[SM_LIST], run[SM_LIST];  // composites as they came, in order; running sums
    u64 wave_sum[SM_WAVES], hit_sum, answer_sum, min_p_sum;
    uint32_t wave_count[SM_WAVES], hit_count, answer_index;
    float wave_top[SM_WAVES];
    int hit, lowest, fill;
};

// sum and count become running sums from bin 0 on.  Whole workgroup; barriers before and after.
__device__ __forceinline__ void running(u64 *sum, uint32_t *count, Shared &s, int tid, int lane, int wave) {
    __syncthreads();
    const u64 a = sum[2 * tid], b = sum[2 * tid + 1];
    const uint32_t ca = count[2 * tid], cb = count[2 * tid + 1];
    u64 w = a + b;
    uint32_t c = ca + cb;
#pragma unroll
    for (int by = 1; by < 64; by <<= 1) {
        const u64 o = __shfl_up(w, by, kWave);
        const uint32_t oc = __shfl_up(c, by, kWave);
        if (lane >= by) {
            w += o;
            c += oc;
        }
    }
    if (lane == 63) {
        s.wave_sum[wave] = w;
        s.wave_count[wave] = c;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < SM_WAVES; ++v)
        if (v < wave) {
            w += s.wave_sum[v];
            c += s.wave_count[v];
        }
    sum[2 * tid] = w - b;
    sum[2 * tid + 1] = w;
    count[2 * tid] = c - cb;
    count[2 * tid + 1] = c;
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

__global__ __launch_bounds__(SM_THREADS) void sample_rows_kernel(const SampleArgs p) {
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x, n = p.n;
    const float *row = p.logits + (size_t)r * n;
    const float temperature = p.temperatures ? p.temperatures[r] : p.temperature, top_p = p.top_ps ? p.top_ps[r] : p.top_p;
    const float min_p = p.min_ps ? p.min_ps[r] : p.min_p, u = p.u[r];
    const int top_k = p.top_ks ? p.top_ks[r] : p.top_k;

    auto for_row = [&](auto &&visit) {  // (i, x) of every element, four in a run
        const int whole = n - n % (4 * SM_THREADS);
#pragma unroll 4
        for (int i = 4 * tid; i < whole; i += 4 * SM_THREADS) {
            const float4 x = load4(row + i);
            visit(i, x.x);
            visit(i + 1, x.y);
            visit(i + 2, x.z);
            visit(i + 3, x.w);
        }
        for (int i = whole + tid; i < n; i += SM_THREADS) visit(i, row[i]);
    };
    float top = -INFINITY;
    for_row([&](int, float x) { top = fmaxf(top, x); });
    top = wave_max(top);
    if (lane == 0) s.wave_top[wave] = top;
    for (int i = tid; i < SM_BINS; i += SM_THREADS) {
        s.sum[i] = 0;
        s.count[i] = 0;
    }
    if (tid == 0) s.min_p_sum = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SM_WAVES; ++w) top = fmaxf(top, s.wave_top[w]);
    if (top == -INFINITY) {  // uniform: nothing to draw from
        if (tid == 0) p.tokens[r] = -1;
        return;
    }
    const Scale scale(top, temperature, p.bits);
    const u64 one = 1ull << p.bits;
    const u64 least = min_p > 0.0f ? (u64)__builtin_ceil(fmin((double)min_p, 2.0) * (double)one) : 0;
    u64 above = 0;  // sum of the weights from min_p on
    for_row([&](int, float x) {
        const double t = scale.log2_of(x);
        if (!scale.counts(t)) return;
        const u64 w = scale.weight(t);
        const int b = scale.bin(t);
        atomicAdd(&s.sum[b], w);
        atomicAdd(&s.count[b], 1u);
        above += w >= least ? w : 0;
    });
    if (min_p > 0.0f) {
#pragma unroll
        for (int by = 32; by > 0; by >>= 1) above += __shfl_xor(above, by, kWave);
        if (lane == 0) atomicAdd(&s.min_p_sum, above);
    }
    running(s.sum, s.count, s, tid, lane, wave);

    // The list: everything of rank list_count0 + 1 to list_count0 + listed, before which the sum is list_sum0.
    u64 list_sum0 = 0;
    uint32_t list_count0 = 0;
    int listed = 0;
    auto fill_list = [&](auto &&takes, u64 sum0, uint32_t count0) {  // takes(t, c): of the list, SM_LIST at most
        if (tid == 0) s.fill = 0;
        __syncthreads();
        for_row([&](int i, float x) {
            const double t = scale.log2_of(x);
            if (!scale.counts(t)) return;
            const u64 c = composite(x, i);
            if (takes(t, c)) s.list[min(atomicAdd(&s.fill, 1), SM_LIST - 1)] = c;
        });
        __syncthreads();
        listed = min(s.fill, SM_LIST);
        list_sum0 = sum0;
        list_count0 = count0;
        if (tid < listed) {  // the place of an element is the number of elements before it
            const u64 mine = s.list[tid];
            int before = 0;
            for (int c = 0; c < listed; ++c) before += s.list[c] > mine ? 1 : 0;
            s.ranked[before] = mine;
        }
        __syncthreads();
        u64 w = tid < listed ? scale.weight(scale.log2_of(value_of(s.ranked[tid]))) : 0;
        if (tid < SM_LIST) {
#pragma unroll
            for (int by = 1; by < 64; by <<= 1) {
                const u64 o = __shfl_up(w, by, kWave);
                if (lane >= by) w += o;
            }
            if (lane == 63) s.wave_sum[wave] = w;
        }
        __syncthreads();
        if (tid < SM_LIST) {
            for (int v = 0; v < wave; ++v) w += s.wave_sum[v];
            s.run[tid] = sum0 + w;
        }
        __syncthreads();
    };
    // the bin of running sums where the target lies, or -1: s.hit, and the sum and count before it
    auto find_bin = [&](const u64 *sum, const uint32_t *count, u64 sum0, uint32_t count0, const Target &to) {
        if (tid == 0) s.hit = -1;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int b = 2 * tid + e;
            const u64 s0 = sum0 + (b ? sum[b - 1] : 0);
            const uint32_t c0 = count0 + (b ? count[b - 1] : 0);
            if (to.within(s0, c0, sum0 + sum[b], count0 + count[b])) {
                s.hit = b;
                s.hit_sum = s0;
                s.hit_count = c0;
            }
        }
        __syncthreads();
        return s.hit;
    };
    // -> s.answer_index and s.answer_sum, the running sum with that rank; false: no such rank
    auto select = [&](const Target &to) {
        __syncthreads();
        const u64 end_sum = listed ? s.run[listed - 1] : 0;
        if (!listed || !to.within(list_sum0, list_count0, end_sum, list_count0 + listed)) {
            const int b = find_bin(s.sum, s.count, 0, 0, to);
            if (b < 0) return false;
            const uint32_t in_bin = s.count[b] - s.hit_count;
            if (in_bin <= SM_LIST) {
                // as many bins before it as there is room for
                if (tid == 0) s.lowest = b;
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = 2 * tid + e;
                    if (c < b && s.count[b] - (c ? s.count[c - 1] : 0) <= SM_LIST) atomicMin(&s.lowest, c);
                }
                __syncthreads();
                const int first = s.lowest;
                fill_list([&](double t, u64) { const int x = scale.bin(t); return x >= first && x <= b; }, first ? s.sum[first - 1] : 0,
                          first ? s.count[first - 1] : 0);
            } else {
                u64 prefix = 0;
                u64 sum0 = s.hit_sum;
                uint32_t count0 = s.hit_count;
                for (int known = 52;;) {  // the bits of a composite; those from `known` on are the same, `prefix`
                    const int shift = max(known - 11, 0);
                    __syncthreads();
                    for (int i = tid; i < SM_BINS; i += SM_THREADS) {
                        s.fine_sum[i] = 0;
                        s.fine_count[i] = 0;
                    }
                    __syncthreads();
                    for_row([&](int i, float x) {
                        const double t = scale.log2_of(x);
                        if (!scale.counts(t) || scale.bin(t) != b) return;
                        const u64 c = composite(x, i);
                        if (c >> known != prefix) return;
                        const int d = SM_BINS - 1 - (int)((c >> shift) & ((1ull << (known - shift)) - 1));
                        atomicAdd(&s.fine_sum[d], scale.weight(t));
                        atomicAdd(&s.fine_count[d], 1u);
                    });
                    running(s.fine_sum, s.fine_count, s, tid, lane, wave);
                    const int d = find_bin(s.fine_sum, s.fine_count, sum0, count0, to);
                    const uint32_t in_piece = s.fine_count[d] - (d ? s.fine_count[d - 1] : 0);
                    sum0 = s.hit_sum;
                    count0 = s.hit_count;
                    prefix = prefix << (known - shift) | (u64)(SM_BINS - 1 - d);
                    known = shift;
                    if (in_piece <= SM_LIST || shift == 0) {
                        fill_list([&](double t, u64 c) { return scale.bin(t) == b && c >> known == prefix; }, sum0, count0);
                        break;
                    }
                }
            }
        }
        if (tid < listed) {
            const u64 before = tid ? s.run[tid - 1] : list_sum0;
            if (to.within(before, list_count0 + tid, s.run[tid], list_count0 + tid + 1)) {
                s.answer_index = (uint32_t)index_of(s.ranked[tid]);
                s.answer_sum = s.run[tid];
            }
        }
        __syncthreads();
        return true;
    };

    const u64 all = s.sum[SM_BINS - 1];
    u64 of_k = all, kept = all;
    if (top_k > 0 && (uint32_t)top_k < s.count[SM_BINS - 1] && select({true, (u64)(top_k - 1)})) of_k = s.answer_sum;
    kept = of_k;
    if (top_p < 1.0f) {
        const double share = (double)top_p * (double)of_k;
        if (share > 0.0) {
            const u64 past = min((u64)__builtin_ceil(share) - 1, of_k - 1);
            if (select({false, past})) kept = min(kept, s.answer_sum);
        } else {
            kept = one;
        }
    }
    if (min_p > 0.0f) kept = min(kept, s.min_p_sum);
    kept = max(kept, one);  // the first is always kept
    const double at = (double)u * (double)kept;
    const u64 past = at > 0.0 ? min((u64)at, kept - 1) : 0;
    select({false, past});
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
    const int bits = std::min(62 - (n > 1 ? 32 - __builtin_clz(n - 1) : 0), 50);
    const SampleArgs p = {logits, u, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p, top_k, tokens_out, n, bits};
    hipLaunchKernelGGL(sample_rows_kernel, dim3(rows), dim3(SM_THREADS), 0, ctx->stream, p);
    return AGPU_LAUNCH_CHECK(ctx, "sample_rows_kernel");
}
