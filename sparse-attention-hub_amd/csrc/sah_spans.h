// Host side: whether an output shares memory with what a call reads, judged by addresses, strides and counts.
#pragma once
#include <stdint.h>

// From a tensor's first byte to behind its last one, judged by strides (elements) and counts
struct sah_span { int64_t lo, hi; };
template <int N>
static inline sah_span sah_span_of(const void* p, int es, int64_t inner, const int64_t (&stride)[N], const int64_t (&count)[N]) {
  sah_span s{0, inner};
  for (int i = 0; i < N; ++i) (stride[i] < 0 ? s.lo : s.hi) += stride[i] * (count[i] - 1);
  return sah_span{(int64_t)(uint64_t)p + s.lo * es, (int64_t)(uint64_t)p + s.hi * es};
}
static inline bool sah_meet(const sah_span& a, const sah_span& b) { return a.lo < b.hi && b.lo < a.hi; }

// Whether a row of out [n_tokens, Hq, D] shares memory with one of q. Where their tokens are equally far apart (two slices of one buffer) every pair of
// heads is looked at: only the nearest tokens can meet. Else tensors that lie within each other count as sharing.
static inline bool sah_out_on_queries(const void* q, int64_t qs_t, int64_t qs_h, const void* out, int64_t os_t, int64_t os_h, int n_tokens, int Hq,
                                      int D, int es) {
  if (!sah_meet(sah_span_of<2>(out, es, D, {os_t, os_h}, {n_tokens, Hq}), sah_span_of<2>(q, es, D, {qs_t, qs_h}, {n_tokens, Hq}))) return false;
  if (os_t != qs_t || Hq > 1024) return true;
  const int64_t first = (int64_t)(uint64_t)out - (int64_t)(uint64_t)q, row = (int64_t)D * es, step = os_t * es;
  for (int ho = 0; ho < Hq; ++ho)
    for (int hq = 0; hq < Hq; ++hq) {
      const int64_t d = first + (ho * os_h - hq * qs_h) * es, near = step ? -d / step : 0;
      for (int64_t i = near - 1; i <= near + 1; ++i)  // tokens that out's row is ahead of q's
        if (i > -n_tokens && i < n_tokens && d + i * step < row && d + i * step > -row) return true;
    }
  return false;
}
