// The next token of each row of logits from one given random number.
//
// In the order of falling logits (ties to the lower index) top-k and top-p both keep a first part, so both are a last kept
// token. Weights are exp((x - m) / t) in fp64, summed as integers of 2^-43: sums of up to 2^20 of them fit 64 bits, are
// exact, and so do not depend on who adds when.
//
// A workgroup has a row. Everything that decides is a selection of one kind: of weighted items in an order, the one at which the
// running weight reaches a target: the k-th largest (weight 1), top-p's last (a token's weight), the drawn token (the same in
// the order of the index). Weights are added up per piece of the order's range in LDS, the few items of the piece that holds the target
// are ranked by a wave (sm_pick). It runs over a list in LDS of all tokens that may be kept, where that can hold them: what may
// be kept is known early, since where r of 1024 threads' own largest logits reach a value, at least r of the row do, and few
// more. Where it cannot, the row is cut into pieces of 1 / SM_FINE in (m - x) / t first, and the list holds one of them.
#include "sah_common.h"
#include "../../include/sah_serve.h"

#define SM_NT 1024
#define SM_NW (SM_NT / SAH_WAVE)
#define SM_ONE 0x1p43
#define SM_MAX_VOCAB (1 << 20)
#define SM_CAP 8192        // tokens of the list
#define SM_BINS 2048
#define SM_SMALL 64        // items that are ranked at once, one a lane
#define SM_FINE 64.f
#define SM_RANK_K 1000     // top-k up to this goes by the threads' largest logits (1024 ln(1024 / 24) = 3800 tokens on average) ...
#define SM_RANK_P 1021     // ... and top-p tries the tokens above this one of them (6000)
#define SM_LOWEST 0x00800000u  // order of the lowest finite logit
typedef sah_u4 sm_vec __attribute__((aligned(2)));

struct sm_shared {
  uint2 list[SM_CAP];         // (float bits, index); or the row's segments' sums
  uint64_t bins[SM_BINS];     // zero between uses
  uint64_t wave_sum[SM_NW];
  uint64_t small_weight[SM_SMALL];
  uint2 small[SM_SMALL];      // (order, index)
  uint64_t found_before;
  int found_bin;
  int n_small[2];
  float wave_max[SM_NW], wave_low[SM_NW];
  int wave_at[SM_NW];
  int count;
};

// order-preserving; equal logits (0 and -0 too) share one
__device__ __forceinline__ uint32_t sm_order(float v) { return sah_sort_key<SAH_F32>(v); }
__device__ __forceinline__ float sm_value(uint32_t order) { return sah_bits_to_float((order & 0x80000000u) ? order ^ 0x80000000u : ~order); }

// a b + c with c in a scalar register. (Left to itself the compiler accumulates onto c, a copy of it for every product.)
__device__ __forceinline__ double sm_fma(double a, double b, double c) {
#if defined(__HIP_DEVICE_COMPILE__)
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
#else
  return a * b + c;
#endif
}
// exp((v - m) / t) = 2^n 2^f, |f| <= 1/2: 2^f by a polynomial of degree 9 (a fit for this interval, off by 1.6e-14 at most). An LDS
// table of 2^(j / 64) and a series of degree 4 instead: 64 lanes' reads meet in the banks, no faster.
struct sm_weights {
  double m, c;             // the largest logit, log2(e) / t
  __device__ __forceinline__ sm_weights(float largest, float t) {
    // +inf is taken as a number so large that all finite ones are far below it, also where t is infinite
    m = largest == INFINITY ? 0x1p1023 : (double)largest;
    c = largest == INFINITY || t == INFINITY ? 1e-300 : 1.4426950408889634 / (double)t;
  }
  __device__ __forceinline__ double operator()(float v) const {
    // (-inf, NaN and what is far below come to 2^-64)
    const double y = fmin(fmax(((double)v - m) * c, -64.0), 0.0);
    const double near = y + 0x1.8p52, n = near - 0x1.8p52, f = y - n;  // the nearest whole number, in the low bits too
    double p = sm_fma(f, 1.0148123730040949e-07, 1.3258333889433935e-06);
    p = sm_fma(f, p, 1.525299113787619e-05);
    p = sm_fma(f, p, 0.0001540344088852882);
    p = sm_fma(f, p, 0.0013333557623583215);
    p = sm_fma(f, p, 0.009618129181165067);
    p = sm_fma(f, p, 0.055504108668426984);
    p = sm_fma(f, p, 0.24022650695722755);
    p = sm_fma(f, p, 0.6931471805598848);
    p = fma(f, p, 1.0);
    return ldexp(p, (int)(uint32_t)__builtin_bit_cast(uint64_t, near));
  }
};
// e to the nearest multiple of 2^-43 (e <= 1), above that of 0
#define SM_ZERO 0x4080000000000000ull  // 512.0
__device__ __forceinline__ uint64_t sm_raw(double e) { return __builtin_bit_cast(uint64_t, e + 512.0); }
__device__ __forceinline__ uint64_t sm_fixed(double e) { return sm_raw(e) - SM_ZERO; }

// sum and exclusive scan over the workgroup's threads (one wait; wave_sum is free to be written when this is called)
__device__ __forceinline__ uint64_t sm_block_scan(uint64_t v, sm_shared& S, uint64_t& all) {
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const uint64_t incl = sah_wave_incl_scan_u64(v);
  if (lane == SAH_WAVE - 1) S.wave_sum[wave] = incl;
  __syncthreads();
  const uint64_t sums = sah_wave_incl_scan_u64(lane < SM_NW ? S.wave_sum[lane] : 0);
  all = sah_lane_u64(sums, SM_NW - 1);
  return (wave ? sah_lane_u64(sums, wave - 1) : 0) + incl - v;
}

// token e of 16 bytes
template <int DT>
__device__ __forceinline__ float sm_unpack(const sah_u4& v, int e) {
  if constexpr (DT == SAH_F32) return sah_bits_to_float(v[e]);
  else if constexpr (DT == SAH_BF16) return sah_bits_to_float(e & 1 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
  else return sah_f16_to_float((uint16_t)(v[e / 2] >> (16 * (e & 1))));
}

// f(logit, index) for every token of the row; a thread meets its own in the order of the index. U: 16-byte pieces a thread
// requests at once; 1: with the next one on its way (where f is long, so that its code is there 16 / ES times, not four times that).
template <int DT, int U, typename F>
__device__ __forceinline__ void sm_each(const void* x, int V, F f) {
  constexpr int ES = DT == SAH_F32 ? 4 : 2, E = 16 / ES;
  auto load = [&](int i) __attribute__((always_inline)) -> sah_u4 { return *(const sm_vec*)((const char*)x + (int64_t)i * ES); };
  const int mine = (int)threadIdx.x * E, step = SM_NT * E;
  auto all_of = [&](const sah_u4& v, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < E; ++e) f(sm_unpack<DT>(v, e), i + e);
  };
  int i = mine;
  if constexpr (U == 1) {
    sah_u4 next = {0, 0, 0, 0};
    if (i + E <= V) next = load(i);
#pragma unroll 1
    for (; i + E <= V; i += step) {
      const sah_u4 v = next;
      if (i + step + E <= V) next = load(i + step);
      all_of(v, i);
    }
  } else {
    for (; i + (U - 1) * step + E <= V; i += U * step) {
      sah_u4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = load(i + u * step);
#pragma unroll
      for (int u = 0; u < U; ++u) all_of(v[u], i + u * step);
    }
#pragma unroll 1
    for (; i + E <= V; i += step) all_of(load(i), i);
  }
#pragma unroll 1
  for (int e = i; e < V && e < i + E; ++e) f(sah_load<DT>(x, e), e);  // the row's last few
}

struct sm_bin {
  int at;            // the bin, -1: the weights do not reach the target
  uint64_t before;   // weight of the bins ahead of it
};
// Adds up what `each` hands to its argument (bin, weight) and finds where the running weight, from bin 0 on, reaches
// target(all the weight). All threads call; ends behind a wait.
template <typename TARGET, typename EACH>
__device__ __forceinline__ sm_bin sm_locate(sm_shared& S, TARGET target_of, EACH each) {
  static_assert(SM_BINS == 2 * SM_NT, "two bins a thread");
  each([&](uint32_t bin, uint64_t weight) { atomicAdd((unsigned long long*)&S.bins[bin], (unsigned long long)weight); });
  if (threadIdx.x == 0) S.found_bin = -1;
  __syncthreads();
  const int b = 2 * (int)threadIdx.x;
  const uint64_t w0 = S.bins[b], w1 = S.bins[b + 1];
  S.bins[b] = 0;
  S.bins[b + 1] = 0;
  uint64_t all;
  const uint64_t before = sm_block_scan(w0 + w1, S, all), target = target_of(all);
  if (before < target && target <= before + w0 + w1) {  // one thread, where the target is reached
    const bool second = before + w0 < target;
    S.found_bin = second ? b + 1 : b;
    S.found_before = second ? before + w0 : before;
  }
  __syncthreads();
  sm_bin r{S.found_bin, S.found_before};
  return r;
}

struct sm_item {
  bool any;
  uint32_t order;
  int index;
};
// Of items (order, index, weight) that `each` hands to its argument, from the largest order down, equal ones by index: the one at
// which the running weight reaches target(all the weight) (> 0). Items outside [lo, hi] are passed over. `round` counts calls.
template <typename TARGET, typename EACH>
__device__ __forceinline__ sm_item sm_pick(sm_shared& S, int& round, uint32_t lo, uint32_t hi, TARGET target_of, EACH each) {
  uint64_t before = 0, target = 0;
  bool first = true;
  bool ties = false;   // all that is left shares one order, `same`: the order is that of the index now
  uint32_t same = 0;
  for (;;) {
    const uint32_t range = hi - lo;
    const int bits = range ? 32 - __builtin_clz(range) : 0, shift = bits > 11 ? bits - 11 : 0;
    auto inside = [&](auto f) __attribute__((always_inline)) {
      each([&](uint32_t order, int index, uint64_t weight) {
        if (ties && order != same) return;
        const uint32_t o = ties ? ~(uint32_t)index : order;
        if (o >= lo && o <= hi) f(o, order, index, weight);
      });
    };
    const sm_bin bin = sm_locate(
        S, [&](uint64_t all) {
          if (first) target = target_of(all);
          return target - before;
        },
        [&](auto put) { inside([&](uint32_t o, uint32_t, int, uint64_t weight) { put((hi - o) >> shift, weight); }); });
    if (bin.at < 0) return sm_item{false, 0, 0};
    first = false;
    before += bin.before;
    hi -= (uint32_t)bin.at << shift;
    lo = hi - lo > (1u << shift) - 1 ? hi - ((1u << shift) - 1) : lo;
    // the piece's items, if they are few
    int* n_small = &S.n_small[round & 1];
    inside([&](uint32_t, uint32_t order, int index, uint64_t weight) {
      const int j = atomicAdd(n_small, 1);
      if (j < SM_SMALL) {
        S.small[j] = make_uint2(order, (uint32_t)index);
        S.small_weight[j] = weight;
      }
    });
    __syncthreads();
    const int n = *n_small;
    if (threadIdx.x == 0) S.n_small[~round & 1] = 0;  // (last read before the waits since)
    ++round;
    if (n <= SM_SMALL) {  // every wave by itself
      const int lane = threadIdx.x & (SAH_WAVE - 1);
      const uint2 me = lane < n ? S.small[lane] : make_uint2(0, 0);
      const uint64_t weight = lane < n ? S.small_weight[lane] : 0;
      uint64_t ahead = before;
      for (int j = 0; j < n; ++j) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)me.x, j), i = (uint32_t)__builtin_amdgcn_readlane((int)me.y, j);
        const uint64_t w = sah_lane_u64(weight, j);
        if (o > me.x || (o == me.x && i < me.y)) ahead += w;
      }
      const uint64_t hit = __ballot(lane < n && ahead < target && target <= ahead + weight);
      const int at = hit ? __builtin_ctzll(hit) : 0;
      return sm_item{hit != 0, (uint32_t)__builtin_amdgcn_readlane((int)me.x, at), __builtin_amdgcn_readlane((int)me.y, at)};
    }
    if (shift == 0 && !ties) {
      ties = true;
      same = lo;
      lo = ~(uint32_t)(SM_MAX_VOCAB - 1);
      hi = ~0u;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(SM_NT, 4) void k_sample(sah_sample_args P) {
  sah_touch_kernargs<sizeof(sah_sample_args)>();
  SAH_DYNAMIC_LDS(s_dyn);
  sm_shared& S = *(sm_shared*)s_dyn;
  constexpr int ES = DT == SAH_F32 ? 4 : 2, E = 16 / ES;
  const int r = blockIdx.x, V = P.vocab;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const void* x = (const char*)P.logits + (int64_t)r * P.row_pitch * ES;
  const float temp = P.temperatures ? P.temperatures[r] : P.temperature;
  const int k = P.top_ks ? P.top_ks[r] : P.top_k;
  const float p = P.top_ps ? P.top_ps[r] : P.top_p;
  float least = P.min_ps ? P.min_ps[r] : P.min_p;
  least = least > 1.f ? 1.f : least;
  const bool use_k = k > 0 && k < V, use_p = p < 1.f, use_m = least > 0.f;
  for (int b = threadIdx.x; b < SM_BINS; b += SM_NT) S.bins[b] = 0;
  if (threadIdx.x == 0) S.count = S.n_small[0] = S.n_small[1] = 0;
  int round = 0;

  // the largest logit and its first place
  float best = -INFINITY;
  int best_at = INT32_MAX;
  sm_each<DT, 4>(x, V, [&](float v, int i) {
    best_at = v > best ? i : best_at;
    best = v > best ? v : best;
  });
  const float own = best;
  float low = best;  // the smallest of the threads' largest
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float o = __shfl_xor(best, d);
    const int oa = __shfl_xor(best_at, d);
    low = fminf(low, __shfl_xor(low, d));
    best_at = o > best ? oa : (o == best && oa < best_at ? oa : best_at);
    best = fmaxf(o, best);
  }
  if (lane == 0) { S.wave_max[wave] = best; S.wave_at[wave] = best_at; S.wave_low[wave] = low; }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SM_NW; ++i) {
    const float o = S.wave_max[i];
    const int oa = S.wave_at[i];
    low = fminf(low, S.wave_low[i]);
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
  const sm_weights weigh(best, temp);
  const uint32_t top = sm_order(best);

  // pieces of 1 / SM_FINE in (m - x) / t, the last one for all that is further down
  const float fine = SM_FINE / temp;
  auto piece = [&](float v) -> int {
    const float d = (best - v) * fine;
    return v == best ? 0 : d < SM_BINS - 1 ? (int)d : SM_BINS - 1;
  };
  // whole numbers before a token are less than p times the sum where they are less than that rounded up; the first is kept
  auto nucleus = [&](uint64_t all) -> uint64_t {
    const double limit = ceil((double)p * (double)all);
    return limit > 1.0 ? (uint64_t)limit : 1;
  };
  // kept: logits above thr, and of those equal to it the ones with an index up to last
  float thr = -INFINITY;
  int last = -1;
  auto kept = [&](float v, int i) { return v > thr || (v == thr && i <= last); };
  int n_list = 0;
  auto enlist = [&](float v, int i) {
    const int n = atomicAdd(&S.count, 1);
    if (n < SM_CAP) S.list[n] = make_uint2(sah_float_to_bits(v), (uint32_t)i);
  };
  auto list_again = [&](auto take) __attribute__((always_inline)) {  // a new list, of the kept tokens that `take` takes; whether it holds them
    if (threadIdx.x == 0) S.count = 0;
    __syncthreads();
    sm_each<DT, 1>(x, V, [&](float v, int i) { if (kept(v, i) && take(v)) enlist(v, i); });
    __syncthreads();
    n_list = S.count;
    return n_list <= SM_CAP;
  };

  // the tokens that may be kept, in a list, where they are not too many
  bool list = false, complete = true;  // complete: the list has every token that min-p keeps
  const bool total = use_p && !use_k && V > SM_CAP;
  uint64_t whole = 0;                  // total: the weight that top-p's last token reaches ...
  sm_bin border{0, 0};                 // ... and its piece
  uint32_t lowest = SM_LOWEST;         // no token of the list is of a lower order
  if ((use_k || use_p || use_m) && (V <= SM_CAP || !use_k || k <= SM_RANK_K)) {
    float from = -INFINITY;
    if (V > SM_CAP) {
      if ((use_k || use_p) && low > -INFINITY) {  // every thread has a logit
        const uint32_t range = top - sm_order(low);
        const int bits = range ? 32 - __builtin_clz(range) : 0, shift = bits > 11 ? bits - 11 : 0;
        const uint64_t rank = use_k ? k : SM_RANK_P;
        const sm_bin b = sm_locate(S, [&](uint64_t) { return rank; }, [&](auto put) { put((top - sm_order(own)) >> shift, 1); });
        const uint32_t down = ((uint32_t)(b.at + 1) << shift) - 1;  // to the lower end of the piece
        from = sm_value(down < range ? top - down : top - range);
        complete = false;
      }
      if (use_m && !use_k) {
        // e >= least where x >= m + t ln(least); a little below that, for the roundings
        const double at = weigh.m + (double)temp * log((double)least);
        const float below = (float)(at - 1e-6 * (fabs(at) + fabs(weigh.m)) - 1e-30);
        if (below > from || !use_p) {
          from = below == below ? below : -INFINITY;
          complete = true;
        }
      }
      if (from > -INFINITY && from < best) lowest = sm_order(from);
    }
    if (total) {
      // the weights' pass shares the row out into pieces too: if top-p's last token lies below the list, its piece is known
      border = sm_locate(
          S, [&](uint64_t all) { return whole = nucleus(all); },
          [&](auto put) __attribute__((always_inline)) {
            sm_each<DT, 1>(x, V, [&](float v, int i) {
              if (v >= from && v > -INFINITY) enlist(v, i);
              put(piece(v), sm_fixed(weigh(v)));
            });
          });
      if (from > -INFINITY && !complete && piece(from) <= border.at) {
        // further down than the list: all down to there, if it holds that
        const float down = best - (border.at + 1.01f) / fine;
        lowest = border.at < SM_BINS - 1 && down > -INFINITY && down < best ? sm_order(down) : SM_LOWEST;
        list_again([&](float v) { return piece(v) <= border.at; });
      }
    } else {
      sm_each<DT, 4>(x, V, [&](float v, int i) { if (v >= from && v > -INFINITY) enlist(v, i); });
    }
    __syncthreads();
    n_list = S.count;
    list = n_list <= SM_CAP;
  }
  auto each = [&](bool from_list, auto f) __attribute__((always_inline)) {
    if (from_list) {
      for (int j = threadIdx.x; j < n_list; j += SM_NT) {
        const uint2 it = S.list[j];
        f(sah_bits_to_float(it.x), (int)it.y);
      }
    } else {
      sm_each<DT, 1>(x, V, f);
    }
  };
  for (int stage = 0; stage < 2; ++stage) {  // top-k, then top-p
    if (stage ? !use_p : !use_k) continue;
    auto weight = [&](float v) -> uint64_t { return stage ? sm_fixed(weigh(v)) : 1; };
    auto target_of = [&](uint64_t all) -> uint64_t { return !stage ? k : total ? whole : nucleus(all); };
    auto items = [&](bool from_list) {
      return [&, from_list](auto put) __attribute__((always_inline)) {
        each(from_list, [&](float v, int i) { if (kept(v, i)) put(sm_order(v), i, weight(v)); });
      };
    };
    sm_item found{false, 0, 0};
    if (list) {
      found = sm_pick(S, round, lowest, top, target_of, items(true));
    } else {
      uint64_t target = whole;
      sm_bin b = border;
      if (!total)
        b = sm_locate(
            S, [&](uint64_t all) { return target = target_of(all); },
            [&](auto put) __attribute__((always_inline)) { each(false, [&](float v, int i) { if (kept(v, i)) put(piece(v), weight(v)); }); });
      if (b.at < 0) continue;
      auto rest = [&](uint64_t) { return target - b.before; };
      if (list_again([&](float v) { return piece(v) == b.at; })) {
        found = sm_pick(S, round, SM_LOWEST, top, rest, items(true));
      } else {  // (thousands of logits in one piece)
        found = sm_pick(S, round, SM_LOWEST, top, rest, [&](auto put) __attribute__((always_inline)) {
          each(false, [&](float v, int i) { if (kept(v, i) && piece(v) == b.at) put(sm_order(v), i, weight(v)); });
        });
      }
    }
    if (found.any) {
      thr = sm_value(found.order);
      last = found.index;
    }
  }
  auto final_weight = [&](float v, int i) -> uint64_t {
    if (!kept(v, i)) return 0;
    const double e = weigh(v);
    return use_m && e < (double)least && v != best ? 0 : sm_fixed(e);
  };
  double u = P.uniforms_f64 ? ((const double*)P.uniforms)[r] : (double)((const float*)P.uniforms)[r];
  u = u > 0.0 ? u : 0.0;
  auto drawn = [&](uint64_t all) -> uint64_t {  // the running weight passes u times all where it reaches this
    const uint64_t t = u < 1.0 ? (uint64_t)(u * (double)all) : all;
    return (t < all ? t : all - 1) + 1;
  };
  auto answer = [&](int i, uint64_t all) {  // one thread
    P.tokens[r] = i;
    if (P.logprobs) P.logprobs[r] = (float)log(weigh(sah_load<DT>(x, i)) * SM_ONE / (double)all);
  };
  if (list) {
    uint64_t all = 0;
    const sm_item f = sm_pick(
        S, round, ~(uint32_t)(V - 1), ~0u, [&](uint64_t a) { all = a; return drawn(a); },
        [&](auto put) __attribute__((always_inline)) { each(true, [&](float v, int i) { put(~(uint32_t)i, i, final_weight(v, i)); }); });
    if (threadIdx.x == 0) answer(f.index, all);
    return;
  }
  // The whole row: the weights of segments of 4 x 64 E tokens; then inside the one that holds the target.
  constexpr int U = 4, SEG = SAH_WAVE * E * U;
  static_assert(SM_MAX_VOCAB / SEG <= SM_NT && SM_NT <= SM_CAP, "a sum a thread");
  uint64_t* segs = (uint64_t*)S.list;
  const int n_segs = (V + SEG - 1) / SEG;
  __syncthreads();  // the list is no longer read
  auto place = [&](int j) { return (wave + j / U * SM_NW) * SEG + (j % U * SAH_WAVE + lane) * E; };  // this lane's j-th piece
  auto load = [&](int i) __attribute__((always_inline)) -> sah_u4 { return i + E <= V ? *(const sm_vec*)((const char*)x + (int64_t)i * ES) : sah_u4{0, 0, 0, 0}; };
  sah_u4 next = load(place(0));
  uint64_t part = 0;
  const bool everything = thr == -INFINITY && !use_m;
#pragma unroll 1
  for (int j = 0; wave + j / U * SM_NW < n_segs; ++j) {
    const sah_u4 v = next;
    const int i = place(j);
    next = load(place(j + 1));
    if (i + E <= V && everything) {
#pragma unroll
      for (int e = 0; e < E; ++e) part += sm_raw(weigh(sm_unpack<DT>(v, e)));
      part -= E * SM_ZERO;
    } else if (i + E <= V) {
#pragma unroll
      for (int e = 0; e < E; ++e) part += final_weight(sm_unpack<DT>(v, e), i + e);
    } else {
#pragma unroll 1
      for (int e = 0; i + e < V; ++e) part += final_weight(sah_load<DT>(x, i + e), i + e);
    }
    if (j % U == U - 1) {
      part = sah_lane_u64(sah_wave_incl_scan_u64(part), SAH_WAVE - 1);
      if (lane == 0) segs[wave + j / U * SM_NW] = part;
      part = 0;
    }
  }
  __syncthreads();
  uint64_t all;
  const uint64_t mine = (int)threadIdx.x < n_segs ? segs[threadIdx.x] : 0;
  uint64_t before = sm_block_scan(mine, S, all);
  const uint64_t target = drawn(all);
  if (before < target && target <= before + mine) {  // one thread
    S.found_bin = threadIdx.x;
    S.found_before = before;
  }
  __syncthreads();
  if (wave) return;
  before = S.found_before;
  int hit = -1;
#pragma unroll 1
  for (int q = 0; q < U; ++q) {
    const int i = S.found_bin * SEG + (q * SAH_WAVE + lane) * E;
    uint64_t w[E], own_sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = i + e < V ? final_weight(sah_load<DT>(x, i + e), i + e) : 0;
      own_sum += w[e];
    }
    const uint64_t incl = sah_wave_incl_scan_u64(own_sum);
    uint64_t ahead = before + incl - own_sum;
    if (ahead < target && target <= ahead + own_sum) {  // one lane of one q
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (ahead < target && target <= ahead + w[e]) hit = i + e;
        ahead += w[e];
      }
    }
    before += sah_lane_u64(incl, SAH_WAVE - 1);
  }
  if (hit >= 0) answer(hit, all);
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
