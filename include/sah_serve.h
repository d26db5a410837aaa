/* Entry points of libsah_mi355.so for serving several requests at once: a key-value cache in pages, attention over it
 * for chunks of new tokens and for single ones, and the choice of the next tokens. The reference serves one request at a
 * time from contiguous caches and answers greedily (adapters/huggingface.py:106-202), so none of these has a counterpart
 * there. Conventions and error codes are sah.h's.
 *
 * The cache: K and V of one layer are n_pages pages of page_size tokens each, addressed by element strides (page, token,
 * head; innermost 1; of a dimension of one entry any number). Request b's token at position p lies in page
 * block_table[b][p / page_size], entry p % page_size; the number page * page_size + entry is its slot. A page number outside
 * [0, n_pages) stands for no page: nothing is read or written there, and the keys it would hold are not there. Several layers
 * share one table.
 *
 * One step: n_tokens rows of new tokens, request after request; request b's are rows cu_new[b] .. cu_new[b + 1] - 1. */
#ifndef SAH_SERVE_H
#define SAH_SERVE_H
#include "sah.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Gives the new tokens of a step their places. Request b holds lens[b] tokens and gets new_lens[b] (negative: 0) more; the
 * pages it needs beyond those it has come off the end of the list free_pages[0 .. *free_count), request after request.
 * A request is granted all its tokens or none: none where lens[b] is negative, where its tokens would not fit into
 * table_width pages or into rows [0, n_tokens) (behind requests that pass those rows also one without new tokens), and, among
 * requests that need pages, from the first on for which the list is too short (a request that needs no page is granted still).
 * Outputs: cu_new [n_requests + 1], the running sum of all new_lens, granted or not, at most n_tokens; positions [n_tokens]
 * (lens[b] + i; 0 behind the last request's rows); slot_map [n_tokens] (-1 for a request that is not granted and behind the
 * last one's rows); granted [n_requests], 0 or 1; kv_lens [n_requests], what attention may see: lens[b] + new_lens[b], or 0
 * for a request that is not granted; lens_out, which may be lens, and free_count_out, which may be free_count; the new pages'
 * entries of block_table. work: 2 * n_requests words. At most 4096 requests and 2^30 tokens. */
typedef struct sah_paged_assign_args {
  const int32_t* new_lens;
  const int32_t* lens;
  int32_t* block_table; int64_t table_pitch; int32_t table_width;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t n_pages;        /* length of free_pages */
  int32_t n_requests, page_size, n_tokens;
  int64_t* slot_map;
  int32_t* positions;
  int32_t* cu_new;
  int32_t* kv_lens;
  uint8_t* granted;
  int32_t* lens_out;
  int32_t* free_count_out;
  int32_t* work;
  void* stream;
} sah_paged_assign_args;
int sah_paged_assign(const sah_paged_assign_args* a);

/* Takes the pages of every request with finished[b] != 0 back: they are appended to free_pages (in the order of requests
 * and of their pages), *free_count grows, lens[b] becomes 0 and the entries of block_table that its length takes -1. An entry
 * below 0 is no page and is not appended; any other number is, whatever it is. Pages that a list of n_pages entries has no room
 * for are lost. work: 2 * n_requests words. */
typedef struct sah_paged_release_args {
  const uint8_t* finished;
  int32_t* lens;
  int32_t* block_table; int64_t table_pitch; int32_t table_width;
  int32_t* free_pages;
  int32_t* free_count;
  int32_t n_pages;
  int32_t n_requests, page_size;
  int32_t* work;
  void* stream;
} sah_paged_release_args;
int sah_paged_release(const sah_paged_release_args* a);

/* Writes row t of keys and values [n_tokens, Hkv, D] to slot slot_map[t] of the cache; a slot outside [0, n_pages *
 * page_size) is passed over. Where two rows name the same slot, which of them it holds afterwards is not defined; rows
 * share no memory with the slots that are written. */
typedef struct sah_paged_store_args {
  const void* k; int64_t ks_t, ks_h;
  const void* v; int64_t vs_t, vs_h;
  void* k_cache; int64_t kcs_p, kcs_t, kcs_h;
  void* v_cache; int64_t vcs_p, vcs_t, vcs_h;
  const int64_t* slot_map;
  int32_t dtype;
  int32_t n_tokens, Hkv, D, n_pages, page_size;
  void* stream;
} sah_paged_store_args;
int sah_paged_store(const sah_paged_store_args* a);

/* Attention of the new tokens over the cache, which holds them already. Row cu_new[b] + i of q stands at position
 * p = kv_lens[b] - (cu_new[b + 1] - cu_new[b]) + i and sees the keys j <= p of its request, with window > 0 those of them with
 * j < sink or j > p - window (the Sink and Local maskers' columns). sinks, optional [Hq]: a logit per head in the softmax's
 * denominator. A row that sees nothing is 0. Rows of q behind the last request's are not read and their output is left as it
 * was. Keys beyond table_width pages are not there; positions, and so windows, go by kv_lens all the same. out [n_tokens, Hq,
 * D]. max_context: about how long the longest request is (0: not known); it decides how work is split, never what is computed.
 * page_size: a power of two; table_width * page_size below 2^31 - 4096. Rows of out share no memory with each other or with
 * what is read (refused, as is an out whose rows lie between those of a cache, or between q's with another qs_t than os_t).
 * Logits, softmax statistics and sums are fp32; the weights of 16-bit types enter the second product as two terms of the type
 * together, or, in longer chunks (tiles of 128 rows), as one.
 * work: sah_paged_attention_work_floats(a) floats, no particular content. */
typedef struct sah_paged_attention_args {
  const void* q; int64_t qs_t, qs_h;
  const void* k; int64_t ks_p, ks_t, ks_h;
  const void* v; int64_t vs_p, vs_t, vs_h;
  const int32_t* block_table; int64_t table_pitch; int32_t table_width;
  const int32_t* kv_lens;
  const int32_t* cu_new;
  const float* sinks;
  int32_t dtype;
  int32_t n_requests, n_tokens, Hq, Hkv, D, n_pages, page_size;
  int32_t max_context, sink, window;
  float scaling;
  void* out; int64_t os_t, os_h;
  float* work; int64_t work_floats;
  void* stream;
} sah_paged_attention_args;
int64_t sah_paged_attention_work_floats(const sah_paged_attention_args* a);
int sah_paged_attention(const sah_paged_attention_args* a);

/* One token per row of logits [n_rows, vocab] from one given number u in [0, 1) per row. With x the row (NaN counts as -inf),
 * m its largest value and t its temperature, token i weighs e_i = exp((x_i - m) / t). In the order of falling x, ties to the
 * lower index: top_k > 0 keeps the first top_k; of those, top_p < 1 keeps a token while what comes before it weighs less than
 * top_p of what top_k kept (the first always); of those, min_p > 0 keeps e_i >= min_p (more than 1 counts as 1; a NaN of these two as off). The token is the first, by
 * index, of the kept ones at which their weights, summed in the order of the index, pass u times their sum; u outside [0, 1)
 * counts as the nearest number inside, NaN as 0. t <= 0 or NaN: the largest logit's token. logprobs, optional: the logarithm of
 * the token's share of the kept weight. A row without a logit above -inf gives token -1, logprob -inf; one with logits
 * of +inf chooses among those. Weights and their sums are held in 64 bits and do not depend on the order of the sums.
 * Each of the four settings is an array of n_rows values or, where that is NULL, one value for all. vocab at most 2^20.
 * work: sah_sample_work_bytes(a) bytes, no particular content, 16-byte aligned: few rows are then shared by several workgroups each;
 * NULL: every row by one. The results are the same. */
typedef struct sah_sample_args {
  const void* logits; int64_t row_pitch;
  int32_t dtype;
  int32_t n_rows, vocab;
  const void* uniforms; int32_t uniforms_f64;   /* float, or double where uniforms_f64 != 0 */
  const float* temperatures; const int32_t* top_ks; const float* top_ps; const float* min_ps;
  float temperature; int32_t top_k; float top_p; float min_p;
  int64_t* tokens;
  float* logprobs;
  void* stream;
  void* work; int64_t work_bytes;               /* optional */
} sah_sample_args;
int64_t sah_sample_work_bytes(const sah_sample_args* a);
int sah_sample_tokens(const sah_sample_args* a);

#ifdef __cplusplus
}
#endif
#endif
