// The KV cache in pages: places in it, what a query sees, and how calls are cut up.  Host and device use the same functions, so that the
// tests of these rules run on the CPU.
//   cache   [n_pages][n_kv_heads][page_size][64], pages page_stride elements apart; a slot is page * page_size + offset
//   tables  [batch][width] page ids: position p of request b is on page tables[b][p / page_size]
#pragma once
#include <cstddef>
#include <cstdint>

#include "../../include/agpu.h"

#ifdef __HIPCC__
#define AGPU_HD __host__ __device__ __forceinline__
#else
#define AGPU_HD inline
#endif

namespace paged {

constexpr int kMaxPageSize = 1 << 20;
constexpr int64_t kMaxPositions = 1 << 30;  // of a request: sums of a few of them fit 32 bits

// n / page_size for 0 <= n < 2^31: with l = ceil(log2 page_size) and mul = floor(2^(31+l) / page_size) + 1, mul * page_size exceeds 2^(31+l) by at most
// 2^l, so that n * mul / 2^(31+l) exceeds the quotient by less than 1 / page_size.
struct PageDiv {
    uint32_t mul;
    int shift, size;
    static PageDiv of(int page_size) {
        int l = 0;
        while ((1 << l) < page_size) ++l;
        return {(uint32_t)(((uint64_t)1 << (31 + l)) / (uint64_t)page_size + 1), 31 + l, page_size};
    }
    AGPU_HD int page(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

// The keys that a query at `pos` of a request of kv_len positions sees, numbered without a gap: number v is key v for the v of the first tokens
// that stay visible (`sinks`), and key v + gap behind them.
struct Visible {
    int sinks, count, gap;
    AGPU_HD int key(int v) const { return v < sinks ? v : v + gap; }
};
// held: positions that the table has pages for.  window 0: none.
AGPU_HD Visible visible(int pos, int kv_len, int held, int window, int sinks) {
    int end = pos < kv_len ? pos + 1 : kv_len;
    end = end < held ? end : held;
    if (pos < 0 || end <= 0) return {0, 0, 0};
    int low = window > 0 && pos + 1 > window ? pos + 1 - window : 0;
    int first = sinks < low ? sinks : low;
    first = first < end ? first : end;
    const int rest = end > low ? end - low : 0;
    return {first, first + rest, low - first};
}

// The keys that rows at the positions pos0 .. pos1 see together, numbered without a gap: number v is key v for the v of the first tokens that stay visible
// (`first`), and key v + gap behind them.  Windows may be as large as 32 bits go, and rows may lie before position 0: compared before subtracted.
struct TileKeys {
    int first, count, gap;
    AGPU_HD int key(int v) const { return v < first ? v : v + gap; }
};
AGPU_HD TileKeys tile_keys(int pos0, int pos1, int held, int window, int sinks) {
    int end = pos1 < held ? pos1 + 1 : held;
    end = end > 0 ? end : 0;
    const int low = window > 0 && pos0 >= window ? pos0 - window + 1 : 0;
    int first = sinks < low ? sinks : low;
    first = first < end ? first : end;
    return {first, first + (end > low ? end - low : 0), low - first};
}
// Which of these numbers the row at `pos` sees.
struct RowKeys {
    int last, low, first;
    AGPU_HD bool sees(int v) const { return v <= last && (v > low || v < first); }
};
AGPU_HD RowKeys row_keys(const TileKeys &tile, int pos, int window, int sinks) {
    const int stay = sinks - tile.gap;
    return {pos - tile.gap, window > 0 && pos >= window ? pos - window - tile.gap : -1, window > 0 && stay > tile.first ? stay : tile.first};
}

// `count` keys over workgroups: about as many runs as there are `run` keys in them, `most` at most, of `keys` each (a multiple of 32; the last ones may be
// empty).  More keys never make fewer runs.
struct RunsOf {
    int runs, keys;
};
AGPU_HD RunsOf runs_of(int count, int run, int most) {
    int runs = (int)(((unsigned)count + (unsigned)run / 2) / (unsigned)run);
    runs = runs < 1 ? 1 : runs > most ? most : runs;
    return {runs, ((count + runs - 1) / runs + 31) & ~31};
}
// A run's length for `work` keys in all (added up over the items) that are to be `fill` runs or so: between `least` and what leaves no item more than `most`.
AGPU_HD int run_for(float work, float fill, int least, int longest, int most) {
    const float even = work / fill;
    int run = even < 1048576.0f ? (int)even : 1048576;
    const int needed = (longest + most - 1) / most;
    run = run > least ? run : least;
    run = run > needed ? run : needed;
    return (run + 31) & ~31;
}

// How many runs an item may have at most: `longest` keys in runs of `least`, partial results of item_bytes each in `space`, a ticket for every item of several.
inline int most_runs(int64_t items, int64_t longest, int64_t least, size_t item_bytes, size_t space, int64_t tickets) {
    int64_t runs = (longest + least - 1) / least;
    runs = runs < 64 ? runs : 64;
    if (items > tickets) runs = 1;
    const int64_t room = items > 0 ? (int64_t)(space / item_bytes) / items : 1;
    runs = runs < room ? runs : room;
    return runs < 1 ? 1 : (int)runs;
}
// The most keys a row can see.
inline int64_t longest_row(int64_t held, int64_t window, int64_t sinks) { return window > 0 && window + sinks < held ? window + sinks : held; }

// ---- what calls are refused: 0, or the error and why --------------------------------------------

struct Refusal {
    int32_t code;
    const char *why;
};
constexpr Refusal kFine = {AGPU_OK, ""};

inline int cache_element_bytes(int32_t type) { return type == AGPU_CACHE_F32 ? 4 : type == AGPU_CACHE_F16 || type == AGPU_CACHE_BF16 ? 2 : 0; }

inline Refusal refuse_cache(uintptr_t k_cache, uintptr_t v_cache, int64_t k_page_stride, int64_t v_page_stride, int32_t n_kv_heads, int32_t n_pages,
                            int32_t page_size, int32_t d_head, int32_t cache_type) {
    const int bytes = cache_element_bytes(cache_type);
    if (d_head != 64) return {AGPU_ERR_SHAPE_MISMATCH, "expected d_head = 64"};
    if (bytes == 0) return {AGPU_ERR_UNSUPPORTED, "the cache's type is none of AGPU_CACHE_F32, AGPU_CACHE_F16, AGPU_CACHE_BF16"};
    if (n_kv_heads <= 0 || n_pages <= 0 || page_size <= 0) return {AGPU_ERR_SHAPE_MISMATCH, "a cache has pages, positions on them and heads"};
    if (page_size > kMaxPageSize || (int64_t)n_pages * page_size > INT32_MAX) return {AGPU_ERR_UNSUPPORTED, "pages of 2^20 positions and caches of 2^31 - 1 slots at most"};
    if ((int64_t)n_kv_heads * page_size > INT32_MAX / 64) return {AGPU_ERR_UNSUPPORTED, "a page of 2^31 elements or more"};
    const int64_t page = (int64_t)n_kv_heads * page_size * 64;
    if (n_pages > 1 && (k_page_stride < page || v_page_stride < page)) return {AGPU_ERR_SHAPE_MISMATCH, "pages overlap"};
    if (k_cache % 16 || v_cache % 16 || (n_pages > 1 && (k_page_stride * bytes % 16 || v_page_stride * bytes % 16)))
        return {AGPU_ERR_UNSUPPORTED, "pages of the cache begin at 16 bytes"};
    return kFine;
}

inline Refusal refuse_attention(int32_t tokens, int32_t batch, int32_t n_heads, int32_t n_kv_heads, int32_t table_width, int32_t page_size,
                                int32_t window, int32_t sinks, bool query_start) {
    if (tokens < 0 || batch < 0 || n_heads <= 0 || n_kv_heads <= 0 || table_width < 0 || window < 0 || sinks < 0)
        return {AGPU_ERR_SHAPE_MISMATCH, "negative sizes"};
    if (n_heads % n_kv_heads) return {AGPU_ERR_SHAPE_MISMATCH, "query heads are a multiple of the K/V heads"};
    if ((int64_t)table_width * page_size > kMaxPositions) return {AGPU_ERR_UNSUPPORTED, "a row of the table stands for 2^30 positions at most"};
    if (!query_start && tokens != batch) return {AGPU_ERR_SHAPE_MISMATCH, "without query_start each request has one row"};
    if ((int64_t)tokens * n_heads >= 1 << 23) return {AGPU_ERR_UNSUPPORTED, "2^23 rows of heads or more"};  // (a launch has less than 2^32 threads)
    return kFine;
}

constexpr int kMaxRequests = 4096;  // of a plan: what it adds up about them lies in LDS

inline Refusal refuse_plan(int32_t batch, int32_t table_width, int32_t stack_size, int32_t page_size, int32_t max_tokens) {
    if (batch < 0 || table_width < 0 || stack_size < 0 || max_tokens < 0) return {AGPU_ERR_SHAPE_MISMATCH, "negative sizes"};
    if (page_size <= 0) return {AGPU_ERR_SHAPE_MISMATCH, "page_size is not positive"};
    if (page_size > kMaxPageSize) return {AGPU_ERR_UNSUPPORTED, "pages of 2^20 positions at most"};
    if (batch > kMaxRequests) return {AGPU_ERR_UNSUPPORTED, "4096 requests at most"};
    if ((int64_t)table_width * page_size > kMaxPositions) return {AGPU_ERR_UNSUPPORTED, "a row of the table stands for 2^30 positions at most"};
    return kFine;
}

inline Refusal refuse_append(int32_t tokens, int32_t n_kv_heads) {
    if (tokens < 0) return {AGPU_ERR_SHAPE_MISMATCH, "negative sizes"};
    if ((int64_t)tokens * n_kv_heads >= 1 << 26) return {AGPU_ERR_UNSUPPORTED, "2^26 rows of heads or more"};  // (a launch has less than 2^32 threads)
    return kFine;
}

}  // namespace paged
