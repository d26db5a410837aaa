// The next token of each row of logits from one given random number.
//
// In the order of falling logits (ties to the lower index) top-k and top-p both keep a first part, so both are a threshold:
// the keys (order-preserving, sah_sort_key) above one value, and of those equal to it the first few by index. Weights are
// exp((x - m) / t) in fp64, summed as integers of 2^-43: sums of up to 2^20 of them fit 64 bits, are exact, and so do not
// depend on who adds when.
#include "sah_common.h"
#include "../../include/sah_serve.h"

#define SM_NT 1024
#define SM_NW (SM_NT / SAH_WAVE)
#define SM_ONE 0x1p43
#define SM_MAX_VOCAB (1 << 20)

template <int DT>
__device__ __forceinline__ uint32_t sm_key(const void* x, int i) {  // 0: not a candidate (-inf, NaN)
  const float f = sah_load<DT>(x, i);
  return f > -INFINITY ? sah_sort_key<SAH_F32>(f) : 0u;
}
__device__ __forceinline__ float sm_value(uint32_t key) { return sah_bits_to_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key); }

// exp(-d / t) of a logit d below the largest; +inf logits count alone
__device__ __forceinline__ double sm_weight(uint32_t key, uint32_t top, double over_t) {
  if (key == top) return 1.0;
  const float m = sm_value(top);
  if (m == INFINITY || key == 0u) return 0.0;
  return exp(((double)sm_value(key) - (double)m) * over_t);
}
__device__ __forceinline__ uint64_t sm_fixed(double e) {  // to the nearest multiple of 2^-43 (e <= 1)
  return __builtin_bit_cast(uint64_t, e + 512.0) - __builtin_bit_cast(uint64_t, 512.0);
}

__device__ __forceinline__ uint64_t sm_block_sum(uint64_t v, uint64_t* s) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d);
  __syncthreads();
  if ((threadIdx.x & (SAH_WAVE - 1)) == 0) s[threadIdx.x / SAH_WAVE] = v;
  __syncthreads();
  uint64_t all = 0;
  for (int i = 0; i < SM_NW; ++i) all += s[i];
  return all;
}

template <int DT>
__global__ __launch_bounds__(SM_NT) void k_sample(sah_sample_args P) {
  __shared__ uint64_t s_sum[SM_NW];
  __shared__ uint64_t s_key[SM_NW];
  const int r = blockIdx.x, V = P.vocab;
  const int es = DT == SAH_F32 ? 4 : 2;
  const void* x = (const char*)P.logits + (int64_t)r * P.row_pitch * es;
  const float temp = P.temperatures ? P.temperatures[r] : P.temperature;
  const int k = P.top_ks ? P.top_ks[r] : P.top_k;
  const float p = P.top_ps ? P.top_ps[r] : P.top_p;
  const float least = P.min_ps ? P.min_ps[r] : P.min_p;
  // the largest logit and its first place: the largest (key, ~index)
  uint64_t best = 0;
  for (int i = threadIdx.x; i < V; i += SM_NT) {
    const uint64_t c = ((uint64_t)sm_key<DT>(x, i) << 32) | (uint32_t)~i;
    best = c > best ? c : best;
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)best, d);
    best = o > best ? o : best;
  }
  if ((threadIdx.x & (SAH_WAVE - 1)) == 0) s_key[threadIdx.x / SAH_WAVE] = best;
  __syncthreads();
  for (int i = 0; i < SM_NW; ++i) best = s_key[i] > best ? s_key[i] : best;
  const uint32_t top = (uint32_t)(best >> 32);
  if (top == 0 || !(temp > 0.f)) {
    if (threadIdx.x == 0) {
      P.tokens[r] = top ? (int64_t)(uint32_t)~(uint32_t)best : -1;
      if (P.logprobs) P.logprobs[r] = top ? 0.f : -INFINITY;
    }
    return;
  }
  const double over_t = 1.0 / (double)temp;
  // (thr, last): kept are keys above thr and, of those equal, the ones with an index up to last
  uint32_t thr = 1;
  int last = V;
  auto kept = [&](uint32_t c, int i) { return c > thr || (c == thr && i <= last); };
  auto count = [&](uint32_t at) {
    uint64_t n = 0;
    for (int i = threadIdx.x; i < V; i += SM_NT) n += sm_key<DT>(x, i) >= at;
    return sm_block_sum(n, s_sum);
  };
  if (k > 0 && k < V) {
    uint32_t at = 0;  // the largest value that at least k keys reach
    for (int bit = 31; bit >= 0; --bit)
      if (count(at | (1u << bit)) >= (uint64_t)k) at |= 1u << bit;
    if (at > 0) {
      const uint64_t rest = k - (at == 0xffffffffu ? 0 : count(at + 1));
      int lo = 0, hi = V - 1;  // the first index with `rest` keys equal to it up to there
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        uint64_t n = 0;
        for (int i = threadIdx.x; i <= mid; i += SM_NT) n += sm_key<DT>(x, i) == at;
        if (sm_block_sum(n, s_sum) >= rest) hi = mid; else lo = mid + 1;
      }
      thr = at;
      last = lo;
    }
  }
  auto mass = [&](uint32_t from, int upto) {  // of the kept keys above `from`, and of those equal with an index up to `upto`
    uint64_t n = 0;
    for (int i = threadIdx.x; i < V; i += SM_NT) {
      const uint32_t c = sm_key<DT>(x, i);
      if (kept(c, i) && (c > from || (c == from && i <= upto))) n += sm_fixed(sm_weight(c, top, over_t));
    }
    return sm_block_sum(n, s_sum);
  };
  if (p < 1.f) {
    const double limit = (double)p * (double)mass(0, 0);
    // the smallest key value whose first token has less than the limit before it
    uint32_t lo = thr, hi = top;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if ((double)mass(mid, -1) < limit) hi = mid; else lo = mid + 1;
    }
    if (!((double)mass(lo, -1) < limit)) lo = top;  // p <= 0 keeps the first alone
    // of the tokens at that value, the last with less than the limit before it: before a token at index i stand those up to i - 1
    int a = 0, z = lo == thr ? last : V - 1;
    while (a < z) {  // the largest i such that mass up to i - 1 < limit
      const int mid = a + (z - a + 1) / 2;
      if ((double)mass(lo, mid - 1) < limit) a = mid; else z = mid - 1;
    }
    // the first of all is kept whatever the limit
    const int first = (int)~(uint32_t)best;
    thr = lo;
    last = lo == top && a < first ? first : a;
  }
  auto weight = [&](int i) -> uint64_t {
    const uint32_t c = sm_key<DT>(x, i);
    if (!kept(c, i)) return 0;
    const double e = sm_weight(c, top, over_t);
    return e < (double)least && c != top ? 0 : sm_fixed(e);
  };
  auto upto = [&](int n) {
    uint64_t s = 0;
    for (int i = threadIdx.x; i < n; i += SM_NT) s += weight(i);
    return sm_block_sum(s, s_sum);
  };
  const uint64_t sum = upto(V);
  double u = P.uniforms_f64 ? ((const double*)P.uniforms)[r] : (double)((const float*)P.uniforms)[r];
  u = u > 0.0 ? u : 0.0;
  uint64_t target = u < 1.0 ? (uint64_t)(u * (double)sum) : sum;
  if (target >= sum) target = sum - 1;
  int lo = 0, hi = V - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (upto(mid + 1) > target) hi = mid; else lo = mid + 1;
  }
  if (threadIdx.x == 0) {
    P.tokens[r] = lo;
    if (P.logprobs) P.logprobs[r] = (float)log(sm_weight(sm_key<DT>(x, lo), top, over_t) * SM_ONE / (double)sum);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
extern "C" int sah_sample_tokens(const sah_sample_args* a) {
  if (!a) return sah_fail(SAH_ENULL, "sah_sample_tokens: args is NULL");
  if (a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16) return sah_fail(SAH_EDTYPE, "sah_sample_tokens: dtype %d", a->dtype);
  if (a->n_rows < 0 || a->vocab <= 0) return sah_fail(SAH_EINVAL, "sah_sample_tokens: n_rows must be >= 0, vocab > 0");
  if (a->vocab > SM_MAX_VOCAB) return sah_fail(SAH_ESHAPE, "sah_sample_tokens: vocab %d; at most %d", a->vocab, SM_MAX_VOCAB);
  if (a->row_pitch < a->vocab && a->n_rows > 1) return sah_fail(SAH_EINVAL, "sah_sample_tokens: row_pitch is less than vocab");
  if (a->n_rows == 0) return SAH_OK;
  if (!a->logits || !a->uniforms || !a->tokens) return sah_fail(SAH_ENULL, "sah_sample_tokens: NULL pointer");
  hipStream_t st = (hipStream_t)a->stream;
  sah_timed timed("k_sample", a->stream);
  if (a->dtype == SAH_F32) hipLaunchKernelGGL(k_sample<SAH_F32>, dim3(a->n_rows), dim3(SM_NT), 0, st, *a);
  else if (a->dtype == SAH_BF16) hipLaunchKernelGGL(k_sample<SAH_BF16>, dim3(a->n_rows), dim3(SM_NT), 0, st, *a);
  else hipLaunchKernelGGL(k_sample<SAH_F16>, dim3(a->n_rows), dim3(SM_NT), 0, st, *a);
  return sah_launch_status("sah_sample_tokens");
}
