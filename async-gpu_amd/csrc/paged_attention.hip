// Attention over a KV cache in pages, d_head = 64: o = softmax(q k / 8) v for the rows of several requests, each over the keys of its own block table.
//
// Two kernels, by what the call says about its rows:
//   tokens <= batch  paged_tokens_kernel: every row by itself on the vector units, which suits one new token a request; the lengths are on the device, so that a
//                    chunk of many rows beside many requests without any comes here too, and reads its keys once a row.  Bound by the bytes of K and V: 64
//                    requests of 4096 keys (32 heads over 8, f16) 102 to 112 us, 4.8 to 5.3 TB/s; with 1 to 4018 keys (80 MB) 28 us, of which 5 are the launch and the way to the
//                    first key; one request of 777 keys, 12 heads, fp32, 6.8, a chain of loads.  The query heads of a K/V head (up to 8) share what is read of it.
//   otherwise        paged_rows_kernel: requests with more than eight rows of heads a K/V head in tiles of 128 rows on the matrix cores, the others as above.  Bound by
//                    the instructions of a tile of 32 keys (some 180 vector ones beside 24 matrix products for a 16-bit cache, 330 and 48 for an fp32 one, two waves
//                    a SIMD), which follow from one another and hardly overlap: 4 chunks of 512 rows over 2048 keys, 16 heads, fp32, 101 us, bf16 or f16 62 to 65; 8 x 256
//                    rows in a window of 1024, bf16, 43 us; a prompt of 2048 rows from the first on, 16 heads, fp32, 81 to 88 us, of 8192, bf16, 424 to 450 (644 where every
//                    workgroup goes through its tiles in the same order).  Two prompts of up to 300 rows and 22 tokens, 25 heads, bf16, 23 us: the way to the first tile and
//                    then one after the other, with 4 % of the cycles in matrix and 23 in vector instructions.
//                    How many runs an item may have follows from the sizes of the arguments, whether or not there are as many rows: with q padded to 2048 rows that step takes
//                    27 us, to 4096 rows 34.
// The softmax goes along the keys in one pass: maximum m, sum l and sum o of weights 2^(s - m), taken again in units of a new maximum where there is one.  Keys are
// cut into runs over workgroups, whose (o, m, l) the last one to finish joins (write-through stores, a ticket; the order of the sum is that of the runs, so that
// results do not depend on who is last).  What has to be known for that, the lengths, is on the device only: a grid of fixed size numbers the runs for itself.
#include "paged_kernels.h"

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
    const PagedAttn p = paged_attn(q, q_token_stride, q_head_stride, k_cache, v_cache, k_page_stride, v_page_stride, block_tables, kv_lens, query_start, o, tokens, batch, n_heads,
                                   n_kv_heads, n_pages, page_size, table_width, window, sinks, ctx->strict_sync);
    const int64_t longest = paged::longest_row(p.held, window, sinks);
    return of_type(cache_type, [&](auto type) { return attention_go<decltype(type), PLAIN>(ctx, p, longest, {}, ctx->workspace, ctx->ws_bytes); });
}
