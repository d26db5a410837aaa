// What the kernels on 8-bit pages and on pages' bounds share: a token's request, elements of e4m3, checks of arguments.
#pragma once
#include "sah_common.h"
#include "sah_spans.h"
#include "../../include/sah_pages.h"

#define PG_MAX_D 256

// bytes of an element
__host__ __device__ constexpr int pg_size(int dtype) { return dtype == SAH_F32 ? 4 : dtype == SAH_E4M3 ? 1 : 2; }

// ---------------------------------------------------------------------------
// elements of e4m3 and their scales
// ---------------------------------------------------------------------------
// 2^e of a scale's byte e + 127 (-110 <= e <= 120, so the number has no subnormal form)
__device__ __forceinline__ float pg_scale(uint32_t byte) { return sah_bits_to_float(byte << 23); }
// of byte i of four
__device__ __forceinline__ float pg_scale_of(uint32_t bytes, int i) { return sah_bits_to_float(((bytes >> (8 * i)) & 0xffu) << 23); }

// Two neighbouring elements of four (the lower pair, or the upper one), times a power of two, as two bf16: exact, one instruction.
template <bool UPPER>
__device__ __forceinline__ uint32_t pg_widen2(uint32_t four, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, scale, UPPER));
#else
  return 0;
#endif
}
__device__ __forceinline__ void pg_widen4(uint32_t four, float scale, float (&o)[4]) {
  const uint32_t lo = pg_widen2<false>(four, scale), hi = pg_widen2<true>(four, scale);
  o[0] = sah_bits_to_float(lo << 16);
  o[1] = sah_bits_to_float(lo & 0xffff0000u);
  o[2] = sah_bits_to_float(hi << 16);
  o[3] = sah_bits_to_float(hi & 0xffff0000u);
}
// element i of a row in storage type T; `scale` counts for SAH_E4M3 alone
template <int T>
__device__ __forceinline__ float pg_element(const void* p, int64_t i, float scale) {
  if constexpr (T == SAH_E4M3) {
    return sah_bits_to_float(pg_widen2<false>(((const uint8_t*)p)[i], scale) << 16);
  } else {
    return sah_load<T>(p, i);
  }
}

// ---------------------------------------------------------------------------
// a token's request
// ---------------------------------------------------------------------------
struct pg_request {
  int b;             // -1: no request has the row
  int begin, n_new;  // its rows
  int kv;            // keys it has
  int64_t base;      // row t stands at position base + t
};
__device__ __forceinline__ pg_request pg_none() { return pg_request{-1, 0, 0, 0, 0}; }
// with begin in [0, n_tokens), begin < end
__device__ __forceinline__ pg_request pg_make(const sah_page_requests& R, int page_size, int b, int begin, int end, int kv) {
  pg_request r;
  const int last = end < R.n_tokens ? end : R.n_tokens, most = R.table_width * page_size;
  r.b = b;
  r.begin = begin;
  r.n_new = last - begin;
  r.kv = kv < 0 ? 0 : (kv < most ? kv : most);
  r.base = (int64_t)kv - end;
  return r;
}
// What all lanes of the wave hold, in scalar registers (doubles are divided in vector ones)
__device__ __forceinline__ int64_t pg_uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// a / b for 0 <= a < 2^53, 0 < b: exact. (The 64-bit division of integers is some 150 instructions.)
__device__ __forceinline__ int64_t pg_div(int64_t a, int64_t b) {
  int64_t q = (int64_t)((double)a / (double)b);
  const int64_t r = a - q * b;
  q -= r < 0;
  q += r >= b;
  return q;
}

// By a whole wave, for a row that all of its lanes ask for: 64 requests are looked at in one trip to memory.
__device__ __forceinline__ pg_request pg_find_by_wave(const sah_page_requests& R, int page_size, int t) {
  const int lane = threadIdx.x & (SAH_WAVE - 1);
  int lo = 0, n = R.n_requests;
  while (n > SAH_WAVE) {
    const int step = (n + SAH_WAVE - 1) / SAH_WAVE;
    const int64_t i = (int64_t)(lane + 1) * step - 1;
    const uint64_t behind = __ballot(R.cu_new[lo + (i < n ? (int)i : n - 1) + 1] > t);
    if (!behind) return pg_none();
    const int from = __builtin_ctzll(behind) * step;  // (at most n - 1: lanes beyond it ask what the last one before asks)
    lo += from;
    n = n - from < step ? n - from : step;
  }
  const int b = lo + (lane < n ? lane : n - 1);
  const int begin = R.cu_new[b], end = R.cu_new[b + 1], kv = R.kv_lens[b];
  const uint64_t has = __ballot(begin >= 0 && begin <= t && t < end);  // (running sums that fall: the first one's)
  if (!has) return pg_none();
  const int at = __builtin_ctzll(has);
  return pg_make(R, page_size, __builtin_amdgcn_readlane(b, at), __builtin_amdgcn_readlane(begin, at), __builtin_amdgcn_readlane(end, at),
                 __builtin_amdgcn_readlane(kv, at));
}

// ---------------------------------------------------------------------------
// host: checks that the entry points share. They change what has no meaning (strides of dimensions of one entry) in a copy.
// ---------------------------------------------------------------------------
static inline int pg_check_cache(sah_page_cache& c, bool with_v, const char* what) {
  if (c.n_pages == 1) c.ks_p = c.vs_p = 0;
  if (c.page_size == 1) c.ks_t = c.vs_t = c.D;
  if (c.Hkv == 1) c.ks_h = c.vs_h = 0;
  if (c.dtype < SAH_F32 || c.dtype > SAH_E4M3) return sah_fail(SAH_EDTYPE, "%s: cache of dtype %d", what, c.dtype);
  if (c.n_pages <= 0 || c.Hkv <= 0) return sah_fail(SAH_EINVAL, "%s: n_pages and Hkv must be > 0", what);
  const int unit = c.dtype == SAH_E4M3 ? 16 : 8;
  if (c.D <= 0 || c.D % unit || c.D > PG_MAX_D) return sah_fail(SAH_ESHAPE, "%s: head_dim %d is not a multiple of %d up to 256", what, c.D, unit);
  if (c.page_size <= 0 || (c.page_size & (c.page_size - 1))) return sah_fail(SAH_ESHAPE, "%s: page_size %d is not a power of two", what, c.page_size);
  if (!c.k || (with_v && !c.v)) return sah_fail(SAH_ENULL, "%s: NULL pointer", what);
  if (c.dtype == SAH_E4M3 && (!c.k_scales || (with_v && !c.v_scales))) return sah_fail(SAH_ENULL, "%s: an 8-bit cache without scales", what);
  if (!with_v) {
    c.v = c.k;
    c.vs_p = c.ks_p; c.vs_t = c.ks_t; c.vs_h = c.ks_h;
    c.v_scales = c.k_scales;
  }
  const int es = pg_size(c.dtype);
  if (((uint64_t)c.k | (uint64_t)c.v | (uint64_t)(es * (c.ks_p | c.ks_t | c.ks_h | c.vs_p | c.vs_t | c.vs_h))) % 16)
    return sah_fail(SAH_EINVAL, "%s: the cache's addresses and strides must be multiples of 16 bytes", what);
  // (four scales of a page are read at once where a page has 16 tokens or more, single ones elsewhere: a layer's of small pages may begin anywhere)
  if (c.dtype == SAH_E4M3 && c.page_size >= 16 && ((uint64_t)c.k_scales | (uint64_t)c.v_scales) % 4)
    return sah_fail(SAH_EINVAL, "%s: scales must be 4-byte aligned", what);
  if (c.ks_t < 0 || c.vs_t < 0 || c.ks_t >= 1 << 26 || c.vs_t >= 1 << 26)  // a few tokens of a page: 32-bit offsets
    return sah_fail(SAH_ESHAPE, "%s: a page's tokens are 2^26 elements or more apart", what);
  return SAH_OK;
}
static inline int pg_check_requests(const sah_page_requests& r, int page_size, bool with_rows, const char* what) {
  if (r.n_requests <= 0 || r.table_width <= 0 || (with_rows && r.n_tokens < 0))
    return sah_fail(SAH_EINVAL, "%s: bad sizes (n_requests %d, table_width %d, n_tokens %d)", what, r.n_requests, r.table_width, r.n_tokens);
  if ((int64_t)r.table_width * page_size > INT32_MAX - 4096) return sah_fail(SAH_ESHAPE, "%s: table_width * page_size passes 2^31 - 4097", what);
  if (r.table_pitch < r.table_width) return sah_fail(SAH_EINVAL, "%s: table_pitch is less than table_width", what);
  if (!r.block_table || !r.kv_lens || (with_rows && !r.cu_new)) return sah_fail(SAH_ENULL, "%s: NULL pointer", what);
  return SAH_OK;
}

// A contiguous tensor of a * b * c elements (more than memory has: as far as addresses go)
static inline sah_span pg_span(const void* p, int64_t a, int64_t b, int64_t c, int es) {
  const double bytes = (double)a * b * c * es;
  return sah_span{(int64_t)(uint64_t)p, bytes < 0x1p62 ? (int64_t)(uint64_t)p + a * b * c * es : INT64_MAX};
}
// Whether an output lies on keys, values (which stand for keys where a call has none) or their scales
static inline bool pg_on_cache(const sah_span& out, const sah_page_cache& c) {
  const int es = pg_size(c.dtype);
  return sah_meet(out, sah_span_of<3>(c.k, es, c.D, {c.ks_p, c.ks_t, c.ks_h}, {c.n_pages, c.page_size, c.Hkv})) ||
         sah_meet(out, sah_span_of<3>(c.v, es, c.D, {c.vs_p, c.vs_t, c.vs_h}, {c.n_pages, c.page_size, c.Hkv})) ||
         (c.dtype == SAH_E4M3 && (sah_meet(out, pg_span(c.k_scales, c.n_pages, c.Hkv, c.page_size, 1)) || sah_meet(out, pg_span(c.v_scales, c.n_pages, c.Hkv, c.page_size, 1))));
}
// ... on the table or the lengths
static inline bool pg_on_requests(const sah_span& out, const sah_page_requests& r, bool with_rows) {
  return sah_meet(out, sah_span_of<1>(r.block_table, 4, r.table_width, {r.table_pitch}, {r.n_requests})) ||
         sah_meet(out, sah_span_of<1>(r.kv_lens, 4, 1, {1}, {r.n_requests})) ||
         (with_rows && sah_meet(out, sah_span_of<1>(r.cu_new, 4, 1, {1}, {r.n_requests + 1})));
}

// Where a context's copy goes. Strides of the outputs in elements. A table, where given, names the copies' pages (of a cache whose pages follow
// each other, as many a request as `length` has, or from page first[b] on): what the attention over a copy goes by; what lies behind a context is left as it is
// then. `lost`, where given with it: a byte for each of pg_load_workgroups() workgroups, whether its request has tokens behind `length`, or no place, or an element that
// is none of the copy's type.
struct pg_load_out {
  void *k, *v;
  int64_t s_b, s_h, s_t;
  int length;
  int32_t* table;
  uint8_t* lost;
  const int32_t* first;
};
int64_t pg_load_workgroups(const sah_page_cache& c, const sah_page_requests& r, int length);  // 0: too many
int pg_load(const sah_page_cache& c, const sah_page_requests& r, int dtype, const pg_load_out& out, void* stream, const char* what);
// Places for the contexts of requests with new tokens, one behind the other: first[b], the first of its pages, and lens[b], its length; where `width` pages of a
// request or `room` in all are not enough -1 and 0 for every request.
int pg_place(const sah_page_requests& r, int page_size, int width, int64_t room, int32_t* first, int32_t* lens, void* stream, const char* what);
