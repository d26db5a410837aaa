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

// A workgroup has a row. Everything that decides is a selection of one kind: of weighted items in an order, the one at which the
// running weight reaches a target (sm_select: a digit at a time, weights added up per digit value in LDS): the k-th largest
// (weight 1), top-p's border (a token's weight), the drawn token (the same in the order of the index). It runs over a list in LDS where that can
// hold every token that may be kept, over the row itself where not. What may be kept is known early: of 1024 threads' own
// largest logits at least r values reach the r-th largest, so at least r of the row do, and few more.
#define SM_CAP 8192        // tokens of the list
#define SM_BINS 2048
#define SM_RANK_K 1000     // top-k up to this goes by the threads' largest logits (1024 ln(1024 / 24) = 3800 tokens on average) ...
#define SM_RANK_P 1021     // ... and top-p tries the tokens above this one of them (6000)
typedef sah_u4 sm_vec __attribute__((aligned(2)));

struct sm_shared {
  uint2 list[SM_CAP];      // (float bits, index); or the row's segments' sums
  uint64_t bins[SM_BINS];
  double table[64];        // 2^(j / 64)
  uint64_t wave_sum[SM_NW];
  uint64_t found[4];
  float wave_max[SM_NW];
  int wave_at[SM_NW];
  int count;
};

// order-preserving, above 0 for every logit above -inf; equal logits (0 and -0 too) share one
__device__ __forceinline__ uint32_t sm_order(float v) { return sah_sort_key<SAH_F32>(v); }
__device__ __forceinline__ float sm_value(uint32_t order) { return sah_bits_to_float((order & 0x80000000u) ? order ^ 0x80000000u : ~order); }

// Weights of a row: exp(-d / t) = 2^(n / 64) * exp(f) with |f| <= ln 2 / 128, exp(f) by its series to the fourth power (off by 4e-14)
struct sm_weights {
  double m, c;             // the largest logit, 64 log2(e) / t
  __device__ __forceinline__ double operator()(const double* table, float v) const {
    // (+inf counts as a finite number, the same in every place; -inf, NaN and what is far below come to 0)
    const double y = fmax((fmin((double)v, 0x1p1000) - m) * c, -4096.0);
    const double n = rint(y);
    const int i = (int)n;
    const double f = (y - n) * 0.010830424696249145;  // ln 2 / 64
    double p = fma(f, 1.0 / 24, 1.0 / 6);
    p = fma(f, p, 0.5);
    p = fma(f, p, 1.0);
    p = fma(f, p, 1.0);
    return ldexp(table[i & 63] * p, i >> 6);
  }
};
__device__ __forceinline__ uint64_t sm_fixed(double e) {  // to the nearest multiple of 2^-43 (e <= 1)
  return __builtin_bit_cast(uint64_t, e + 512.0) - __builtin_bit_cast(uint64_t, 512.0);
}

__device__ __forceinline__ uint64_t sm_wave_sum(uint64_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d);
  return v;
}
__device__ __forceinline__ uint64_t sm_block_sum(uint64_t v, sm_shared& S) {
  v = sm_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & (SAH_WAVE - 1)) == 0) S.wave_sum[threadIdx.x / SAH_WAVE] = v;
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (int i = 0; i < SM_NW; ++i) all += S.wave_sum[i];
  return all;
}
// exclusive scan over the workgroup's threads
__device__ __forceinline__ uint64_t sm_block_scan(uint64_t v, sm_shared& S) {
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  uint64_t incl = v;
#pragma unroll
  for (int d = 1; d < SAH_WAVE; d <<= 1) {
    const uint64_t up = __shfl_up((unsigned long long)incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == SAH_WAVE - 1) S.wave_sum[wave] = incl;
  __syncthreads();
  uint64_t before = 0;
#pragma unroll
  for (int i = 0; i < SM_NW; ++i) before += i < wave ? S.wave_sum[i] : 0;
  return before + incl - v;
}

// token e of 16 bytes
template <int DT>
__device__ __forceinline__ float sm_unpack(const sah_u4& v, int e) {
  if constexpr (DT == SAH_F32) return sah_bits_to_float(v[e]);
  else if constexpr (DT == SAH_BF16) return sah_bits_to_float(e & 1 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
  else return sah_f16_to_float((uint16_t)(v[e / 2] >> (16 * (e & 1))));
}

// f(logit, index) for every token of the row; a thread meets its own in the order of the index
template <int DT, typename F>
__device__ __forceinline__ void sm_each(const void* x, int V, F f) {
  constexpr int E = DT == SAH_F32 ? 4 : 8, U = 4;
  constexpr int ES = DT == SAH_F32 ? 4 : 2;
  for (int base = 0; base < V; base += SM_NT * E * U) {
    sah_u4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + (u * SM_NT + (int)threadIdx.x) * E;
      if (i + E <= V) v[u] = *(const sm_vec*)((const char*)x + (int64_t)i * ES);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + (u * SM_NT + (int)threadIdx.x) * E;
      if (i >= V) break;
      if (i + E <= V) {
#pragma unroll
        for (int e = 0; e < E; ++e) f(sm_unpack<DT>(v[u], e), i + e);
      } else {
        for (int e = 0; i + e < V; ++e) f(sah_load<DT>(x, i + e), i + e);
      }
    }
  }
}

struct sm_found {
  bool any;          // the weights reach the target
  uint32_t at;       // the order of the item at which they do
  uint64_t before;   // weight of the items above it
  uint64_t here;     // weight of the items of this order
};
// Of items (order, weight) that `each` hands to its argument, from the largest order down: where the running weight reaches
// `target` (> 0). Orders differ in BITS leading bits, at most. All threads call.
template <int BITS, typename EACH>
__device__ __forceinline__ sm_found sm_select(sm_shared& S, uint64_t target, EACH each) {
  sm_found r{true, 0, 0, 0};
  uint32_t known = 0;  // the leading bits that are decided
  for (int done = 0; done < BITS;) {
    const int bits = BITS - done < 11 ? BITS - done : 11;
    const int shift = 32 - done - bits;
    const uint32_t digit = (1u << bits) - 1;
    for (int b = threadIdx.x; b < SM_BINS; b += SM_NT) S.bins[b] = 0;
    __syncthreads();
    each([&](uint32_t order, uint64_t weight) {
      if ((order & known) == r.at) atomicAdd((unsigned long long*)&S.bins[(order >> shift) & digit], (unsigned long long)weight);
    });
    __syncthreads();
    // a thread's two digit values, from the largest down
    static_assert(SM_BINS == 2 * SM_NT, "two a thread");
    const int b = SM_BINS - 1 - 2 * (int)threadIdx.x;
    const uint64_t w1 = S.bins[b], w0 = S.bins[b - 1];
    const uint64_t before = r.before + sm_block_scan(w1 + w0, S);
    if (threadIdx.x == 0) S.found[0] = 0;
    __syncthreads();
    if (before < target && target <= before + w1 + w0) {  // at most one thread
      const bool second = before + w1 < target;
      S.found[0] = 1;
      S.found[1] = (uint64_t)(second ? b - 1 : b);
      S.found[2] = second ? before + w1 : before;
      S.found[3] = second ? w0 : w1;
    }
    __syncthreads();
    if (!S.found[0]) {
      r.any = false;
      return r;
    }
    r.at |= (uint32_t)S.found[1] << shift;
    r.before = S.found[2];
    r.here = S.found[3];
    known |= digit << shift;
    done += bits;
  }
  return r;
}

template <int DT>
__global__ __launch_bounds__(SM_NT, 4) void k_sample(sah_sample_args P) {
  sah_touch_kernargs<sizeof(sah_sample_args)>();
  SAH_DYNAMIC_LDS(s_dyn);
  sm_shared& S = *(sm_shared*)s_dyn;
  constexpr int ES = DT == SAH_F32 ? 4 : 2, E = 16 / ES;
  constexpr int BITS = DT == SAH_F32 ? 32 : 16 + (DT == SAH_F16 ? 3 : 0);  // fp16 as fp32: 13 of the 23 mantissa bits are 0 (or 1)
  const int r = blockIdx.x, V = P.vocab;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const void* x = (const char*)P.logits + (int64_t)r * P.row_pitch * ES;
  const float temp = P.temperatures ? P.temperatures[r] : P.temperature;
  const int k = P.top_ks ? P.top_ks[r] : P.top_k;
  const float p = P.top_ps ? P.top_ps[r] : P.top_p;
  float least = P.min_ps ? P.min_ps[r] : P.min_p;
  least = least > 1.f ? 1.f : least;
  const bool use_k = k > 0 && k < V, use_p = p < 1.f, use_m = least > 0.f;
  if (threadIdx.x < 64) S.table[threadIdx.x] = exp2(threadIdx.x / 64.0);
  if (threadIdx.x == 0) S.count = 0;

  // the largest logit and its first place
  float best = -INFINITY;
  int best_at = INT32_MAX;
  sm_each<DT>(x, V, [&](float v, int i) {
    best_at = v > best ? i : best_at;
    best = v > best ? v : best;
  });
  const float own = best;
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float o = __shfl_xor(best, d);
    const int oa = __shfl_xor(best_at, d);
    best_at = o > best ? oa : (o == best && oa < best_at ? oa : best_at);
    best = fmaxf(o, best);
  }
  if (lane == 0) { S.wave_max[wave] = best; S.wave_at[wave] = best_at; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SM_NW; ++i) {
    const float o = S.wave_max[i];
    const int oa = S.wave_at[i];
    best_at = o > best ? oa : (o == best && oa < best_at ? oa : best_at);
    best = fmaxf(o, best);
  }
  if (best == -INFINITY || !(temp > 0.f)) {
    if (threadIdx.x == 0) {
      P.tokens[r] = best == -INFINITY ? -1 : best_at;
      if (P.logprobs) P.logprobs[r] = best == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const sm_weights weigh{fmin((double)best, 0x1p1000), 92.33248261893676 / (double)temp};  // 64 log2(e)
  auto fixed = [&](float v) -> uint64_t { return v > -INFINITY ? sm_fixed(weigh(S.table, v)) : 0; };

  // the tokens that may be kept, in a list, where they are not too many
  bool list = false, complete = true;  // complete: the list has every token that min-p keeps
  const bool total = use_p && !use_k && V > SM_CAP;
  uint64_t sum = 0;                    // total: of all weights
  if ((use_k || use_p || use_m) && (V <= SM_CAP || !use_k || k <= SM_RANK_K)) {
    float from = -INFINITY;
    if (V > SM_CAP) {
      if (use_k || use_p) {
        const uint64_t rank = use_k ? k : SM_RANK_P;
        const sm_found f = sm_select<22>(S, rank, [&](auto put) { if (own > -INFINITY) put(sm_order(own), 1); });
        if (f.any) {  // (all values with these 22 bits: the smallest of them)
          from = f.at > 0x007fffffu ? sm_value(f.at) : -INFINITY;  // (0x007fffff: the order of -inf)
          complete = false;
        }
      }
      if (use_m && !use_k) {
        // e >= least where x >= m + t ln(least); a little below that, for the roundings
        const double at = weigh.m + (double)temp * log((double)least);
        const float low = (float)(at - 1e-6 * (fabs(at) + fabs(weigh.m)) - 1e-30);
        if (low > from || !use_p) {
          from = low == low ? low : -INFINITY;
          complete = true;
        }
      }
    }
    uint64_t mine = 0;
    sm_each<DT>(x, V, [&](float v, int i) {
      if (v >= from && v > -INFINITY) {
        const int n = atomicAdd(&S.count, 1);
        if (n < SM_CAP) S.list[n] = make_uint2(sah_float_to_bits(v), (uint32_t)i);
      }
      if (total) mine += fixed(v);
    });
    if (total) sum = sm_block_sum(mine, S);
    __syncthreads();
    list = S.count <= SM_CAP;
  }
  const int n_list = list ? S.count : 0;
  // kept: of a higher order than thr, and of those that share it the ones with an index up to last
  uint32_t thr = 0;
  int last = V;
  auto kept = [&](float v, int i) {
    const uint32_t o = sm_order(v);
    return v > -INFINITY && (o > thr || (o == thr && i <= last));
  };
  auto each = [&](auto f) __attribute__((always_inline)) {
    if (list) {
      for (int j = threadIdx.x; j < n_list; j += SM_NT) {
        const uint2 it = S.list[j];
        f(sah_bits_to_float(it.x), (int)it.y);
      }
    } else {
      sm_each<DT>(x, V, f);
    }
  };
  // the orders of 16-bit types differ in their leading bits alone, the others are 0, of negative numbers 1
  auto whole_order = [&](uint32_t o) { return BITS < 32 && !(o & 0x80000000u) ? o | (uint32_t)((1ull << (32 - BITS)) - 1) : o; };
  // of those that share thr, the first n by index
  auto first_of = [&](uint64_t n) {
    const sm_found f = sm_select<20>(S, n, [&](auto put) {
      each([&](float v, int i) { if (sm_order(v) == thr && kept(v, i)) put(~((uint32_t)i << 12), 1); });
    });
    if (f.any) last = (int)(~f.at >> 12);
  };
  if (use_k) {
    const sm_found f = sm_select<BITS>(S, k, [&](auto put) { each([&](float v, int i) { if (v > -INFINITY) put(sm_order(v), 1); }); });
    if (f.any) {
      thr = whole_order(f.at);
      if (f.before + f.here > (uint64_t)k) first_of(k - f.before);
    }
  }
  if (use_p) {
    if (!total) {
      uint64_t mine = 0;
      each([&](float v, int i) { if (kept(v, i)) mine += fixed(v); });
      sum = sm_block_sum(mine, S);
    }
    // whole numbers before a token are less than p times the sum where they are less than that rounded up
    const double limit = ceil((double)p * (double)sum);
    const uint64_t target = limit > 1.0 ? (uint64_t)limit : 1;  // (the first is always kept)
    auto border = [&]() {
      return sm_select<BITS>(S, target, [&](auto put) { each([&](float v, int i) { if (kept(v, i)) put(sm_order(v), fixed(v)); }); });
    };
    sm_found f = border();
    if (!f.any && list && !complete) {  // the list ends before: the whole row
      list = false;
      f = border();
    }
    if (f.any) {
      const uint32_t at = whole_order(f.at);
      if (at != thr) last = V;
      thr = at;
      const uint64_t e = fixed(sm_value(at));
      const uint64_t n = (target - f.before + e - 1) / e;  // (e > 0: the weight at `at` reaches the target)
      if (n * e < f.here) first_of(n);
    }
  }
  auto final_weight = [&](float v, int i) -> uint64_t {
    if (!kept(v, i)) return 0;
    const double e = weigh(S.table, v);
    return use_m && e < (double)least ? 0 : sm_fixed(e);
  };
  double u = P.uniforms_f64 ? ((const double*)P.uniforms)[r] : (double)((const float*)P.uniforms)[r];
  u = u > 0.0 ? u : 0.0;
  auto target_of = [&](uint64_t all) {
    const uint64_t t = u < 1.0 ? (uint64_t)(u * (double)all) : all;
    return t < all ? t : all - 1;
  };
  auto answer = [&](int i, uint64_t all) {  // one thread
    P.tokens[r] = i;
    if (P.logprobs) P.logprobs[r] = (float)log(weigh(S.table, sah_load<DT>(x, i)) * SM_ONE / (double)all);
  };
  if (list) {
    uint64_t mine = 0;
    each([&](float v, int i) { mine += final_weight(v, i); });
    const uint64_t all = sm_block_sum(mine, S);
    const sm_found f = sm_select<20>(S, target_of(all) + 1, [&](auto put) {
      each([&](float v, int i) { put(~((uint32_t)i << 12), final_weight(v, i)); });
    });
    if (threadIdx.x == 0) answer((int)(~f.at >> 12), all);
    return;
  }
  // The whole row: the weights of segments of 64 E tokens, what a wave reads at once; then inside the one that holds the target.
  constexpr int SEG = SAH_WAVE * E, U = 4;
  static_assert(SM_MAX_VOCAB / SEG <= 4 * SM_NT && 4 * SM_NT <= SM_CAP, "four sums a thread");
  uint64_t* segs = (uint64_t*)S.list;
  const int n_segs = (V + SEG - 1) / SEG;
  auto lane_weights = [&](int seg, uint64_t (&w)[E]) __attribute__((always_inline)) {
    const int i = seg * SEG + lane * E;
    sah_u4 v = {0, 0, 0, 0};
    const bool full = i + E <= V;
    if (full) v = *(const sm_vec*)((const char*)x + (int64_t)i * ES);
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = full ? final_weight(sm_unpack<DT>(v, e), i + e) : i + e < V ? final_weight(sah_load<DT>(x, i + e), i + e) : 0;
  };
  __syncthreads();  // the list is no longer read
  for (int s0 = wave; s0 < 4 * SM_NT; s0 += SM_NW * U) {
    if (s0 >= n_segs) {
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (lane == 0) segs[s0 + q * SM_NW] = 0;
      continue;
    }
    sah_u4 v[U];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int i = (s0 + q * SM_NW) * SEG + lane * E;
      v[q] = sah_u4{0, 0, 0, 0};
      if (i + E <= V) v[q] = *(const sm_vec*)((const char*)x + (int64_t)i * ES);
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int seg = s0 + q * SM_NW, i = seg * SEG + lane * E;
      uint64_t mine = 0;
      if (i + E <= V) {
#pragma unroll
        for (int e = 0; e < E; ++e) mine += final_weight(sm_unpack<DT>(v[q], e), i + e);
      } else {
        for (int e = 0; i + e < V; ++e) mine += final_weight(sah_load<DT>(x, i + e), i + e);
      }
      mine = sm_wave_sum(mine);
      if (lane == 0) segs[seg] = mine;
    }
  }
  __syncthreads();
  uint64_t four[4], mine = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    four[q] = segs[4 * threadIdx.x + q];
    mine += four[q];
  }
  const uint64_t all = sm_block_sum(mine, S);
  const uint64_t target = target_of(all);
  __syncthreads();  // sums of waves are read
  uint64_t before = sm_block_scan(mine, S);
  if (before <= target && target < before + mine) {  // one thread
    int q = 0;
    for (; q < 3 && before + four[q] <= target; ++q) before += four[q];
    S.found[0] = 4 * threadIdx.x + q;
    S.found[1] = before;
  }
  __syncthreads();
  if (wave) return;
  const int seg = (int)S.found[0];
  uint64_t w[E], own_sum = 0;
  lane_weights(seg, w);
#pragma unroll
  for (int e = 0; e < E; ++e) own_sum += w[e];
  uint64_t incl = own_sum;
#pragma unroll
  for (int d = 1; d < SAH_WAVE; d <<= 1) {
    const uint64_t up = __shfl_up((unsigned long long)incl, d);
    if (lane >= d) incl += up;
  }
  before = S.found[1] + incl - own_sum;
  if (before <= target && target < before + own_sum) {  // one lane
    int e = 0;
    for (; before + w[e] <= target; ++e) before += w[e];
    answer(seg * SEG + lane * E + e, all);
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
  auto kernel = a->dtype == SAH_F32 ? k_sample<SAH_F32> : a->dtype == SAH_BF16 ? k_sample<SAH_BF16> : k_sample<SAH_F16>;
  if (int rc = sah_allow_lds((const void*)kernel, sizeof(sm_shared), "sah_sample_tokens")) return rc;
  sah_timed timed("k_sample", a->stream);
  hipLaunchKernelGGL(kernel, dim3(a->n_rows), dim3(SM_NT), sizeof(sm_shared), st, *a);
  return sah_launch_status("sah_sample_tokens");
}
