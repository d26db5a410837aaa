/* Entry points of libsah_mi355.so for a paged cache (sah_serve.h) that is held in 8 bits, and for attention over the pages that matter to
 * a token. The reference's caches are contiguous and in the model's type; its QuestTopKMasker (maskers/fixed/implementations/quest_top_k.py:58) takes pages
 * by the smallest and largest elements of their keys into a mask over a contiguous cache. That score was published as Quest (Tang et al., 2024); here it is summed
 * over the query heads that share a key head, and pages that are not selected are not read.
 * Conventions and error codes are sah.h's, what a cache, a table, a slot and a step are is sah_serve.h's.
 *
 * Eight bits: an element is a number of e4m3 (4 bits of exponent, 3 of mantissa, NaN but no infinity; torch.float8_e4m3fn) times
 * 2^e, e the same for all of a token's elements of one key head: the least whole number from -110 up at which the row's
 * largest finite magnitude is at most 448 * 2^e. The scale is held as the byte e + 127 (torch.float8_e8m0fnu), scales [n_pages, Hkv, page_size].
 * A power of two divides and multiplies exactly: an element is rounded once, to the nearest, ties to even, and what it stands
 * for is a bf16 number; but magnitudes from 248 * 2^120 (3.297e38) on are rounded to 2^128, which bf16 and fp32 do not have, and count as infinite wherever
 * they are read. An element that is not finite is held as NaN. */
#ifndef SAH_PAGES_H
#define SAH_PAGES_H
#include "sah_serve.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SAH_E4M3 3   /* beside sah.h's SAH_F32, SAH_BF16, SAH_F16, where a cache's type is meant */

/* One layer's pages. Addresses and strides (elements; innermost 1; of a dimension of one entry any number) are multiples of 16 bytes, D a
 * multiple of 8 (SAH_E4M3: of 16) up to 256, page_size a power of two, a page's tokens less than 2^26 elements apart. */
typedef struct sah_page_cache {
  void* k; int64_t ks_p, ks_t, ks_h;
  void* v; int64_t vs_p, vs_t, vs_h;
  uint8_t* k_scales;       /* SAH_E4M3: [n_pages, Hkv, page_size], from a page_size of 16 on 4-byte aligned; else not looked at */
  uint8_t* v_scales;
  int32_t dtype;
  int32_t n_pages, page_size, Hkv, D;
} sah_page_cache;

/* Whose pages, and the rows of new tokens: sah_paged_attention's fields of the same names. table_width * page_size is less than 2^31 - 4096. */
typedef struct sah_page_requests {
  const int32_t* block_table; int64_t table_pitch; int32_t table_width;
  const int32_t* kv_lens;
  const int32_t* cu_new;
  int32_t n_requests, n_tokens;
} sah_page_requests;

/* Quantises row t of keys and values [n_tokens, Hkv, D] (dtype) into slot slot_map[t] of a SAH_E4M3 cache, the scales with it. Slots outside the cache
 * are passed over; two rows of one slot: what it holds is not defined (elements of one, the scale of the other). Rows and slots share no memory with the cache. */
typedef struct sah_page_store_args {
  sah_page_cache cache;
  const void* k; int64_t ks_t, ks_h;
  const void* v; int64_t vs_t, vs_h;
  const int64_t* slot_map;
  int32_t dtype;
  int32_t n_tokens;
  void* stream;
} sah_page_store_args;
int sah_page_store(const sah_page_store_args* a);

/* Reads requests' contexts back: k_out and v_out [n_requests, Hkv, length, D] (contiguous) hold the tokens at positions below kv_lens[b], and 0 from
 * there on and on pages that are not there. dtype: the cache's, or for SAH_E4M3 any of the three; SAH_F16 then ends at its
 * largest number, +-65504. Of `requests` cu_new and n_tokens are not looked at. k_out and v_out share no memory with each other or with what is read (refused). */
typedef struct sah_page_load_args {
  sah_page_cache cache;
  sah_page_requests requests;
  void* k_out;
  void* v_out;
  int32_t dtype;
  int32_t length;
  void* stream;
} sah_page_load_args;
int sah_page_load(const sah_page_load_args* a);

/* Bounds [n_pages, Hkv, 2, D] (contiguous; the cache's type, for SAH_E4M3 bf16, which holds them exactly): the smallest and, behind it, the largest
 * element of each channel of a page's keys, NaN where one of them is. Brings those of the pages that the step has filled up to date: pages whose last
 * token is one of the cu_new[b + 1] - cu_new[b] last ones of kv_lens[b]. All others stay as they were. Keys have been written before; v, its strides and scales
 * and n_tokens are not looked at. Bounds share no memory with what is read (refused). */
typedef struct sah_page_bounds_args {
  sah_page_cache cache;
  sah_page_requests requests;
  void* bounds;
  void* stream;
} sah_page_bounds_args;
int sah_page_bounds(const sah_page_bounds_args* a);

/* The pages that a token attends to, for each key head h: of those at or before its own position's page, which are its candidates,
 * the first sink_pages and the last window_pages (its own is the last one), and of the others, up to n_select in all, those of the largest
 *     score(page) = sum over h's query heads and over channels c of max(q_c * smallest_c, q_c * largest_c),
 * ties to the lower page. (What is summed over c is the largest q . k that a key of the page can reach. An infinite bound counts where its product is the larger
 * one; 0 times it is no number.) Scores are held in 64 bits and summed in
 * an order that D and the bounds' type fix: equal bounds score the same and results repeat; scores that are closer to each other than some 4 D * 2^-53 of the sum of
 * their terms' sizes may rank either way. One that is not finite ranks above all others. Pages that the table does not have are no
 * candidates. pages [n_tokens, Hkv, n_select]: places in the request's row of the table, rising, -1 behind the last; -1 alone for rows behind the
 * last request's. Only bounds of candidates that are not taken anyway are read. sink_pages + window_pages <= n_select, window_pages >= 1.
 * Addresses and strides of q and bounds are multiples of 16 bytes; pages share no memory with what is read (refused). max_context: as for sah_paged_attention. work: sah_page_select_work_bytes(a) bytes
 * (8 a token, key head and entry of the table, up to 256 MiB or a single row's), 16-byte aligned, no particular content. */
typedef struct sah_page_select_args {
  const void* q; int64_t qs_t, qs_h;
  const void* bounds;
  int32_t dtype;            /* of q */
  int32_t bounds_dtype;
  int32_t Hq, Hkv, D, n_pages, page_size;
  sah_page_requests requests;
  int32_t n_select, sink_pages, window_pages, max_context;
  int32_t* pages;
  void* work; int64_t work_bytes;
  void* stream;
} sah_page_select_args;
int64_t sah_page_select_work_bytes(const sah_page_select_args* a);
int sah_page_select(const sah_page_select_args* a);

/* sah_paged_attention where the cache is in 8 bits (dtype: of q and out, any of the three), or where pages [n_tokens, Hkv, n_select] names the pages
 * that a token's query heads of a key head attend to (any cache type; else dtype is the cache's). An entry of pages is a place in the request's row of
 * the table; one outside it, or whose page is not there, stands for nothing, and a page that is named twice counts twice. Keys behind a token's own
 * position are hidden also on the pages that are named. With pages there is no window. All else is as there, sinks, rows without a key, rows behind the last
 * request's and what out may share memory with. A row that comes out not finite is done again key by key.
 * Logits, softmax statistics and sums are fp32; q of more than bf16's bits and weights enter 16-bit products as several terms: as
 * exact as the result's own rounding. Chunks of an 8-bit cache under 16-bit q (more than 128 rows of q a request
 * and key head on average, with a window as many times more as the table has keys beyond it) are attended to through a
 * copy in q's type, in work, of the contexts of requests with new tokens, by sah_paged_attention's kernels and with what it says of weights. The copy has room for
 * the table's tokens of every request up to 256 MiB, else max_context ones (0: the table's), or, where this passes 2 GiB, for as many tokens as the cache or 2 GiB hold. Where a context is
 * longer, all of them need more room (requests that share pages), or the cache holds what SAH_F16 does not (beyond 65504, finer than 2^-24), it is attended to as it is
 * all the same. work: sah_page_attention_work_bytes(a) bytes, 16-byte aligned, no particular content. */
typedef struct sah_page_attention_args {
  const void* q; int64_t qs_t, qs_h;
  sah_page_cache cache;
  sah_page_requests requests;
  const int32_t* pages; int32_t n_select;   /* NULL, 0: all pages */
  const float* sinks;
  int32_t dtype;
  int32_t Hq;
  int32_t max_context, sink, window;
  float scaling;
  void* out; int64_t os_t, os_h;
  void* work; int64_t work_bytes;
  void* stream;
} sah_page_attention_args;
int64_t sah_page_attention_work_bytes(const sah_page_attention_args* a);
int sah_page_attention(const sah_page_attention_args* a);

#ifdef __cplusplus
}
#endif
#endif
