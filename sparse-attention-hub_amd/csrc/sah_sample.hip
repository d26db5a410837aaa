// The next token of each row of logits from one given random number.
//
// In the order of falling logits (ties to the lower index) top-k and top-p both keep a first part, so both are a last kept
// token. Weights are exp((x - m) / t) in fp64, summed as integers of 2^-43: sums of up to 2^20 of them fit 64 bits, are
// exact, and so do not depend on who adds when.
//
// A workgroup has a row (few long rows: several, for the passes over all of it). Everything that decides is a selection of one kind: of weighted items in an order, the one at which the
// running weight reaches a target: the k-th largest (weight 1), top-p's last (a token's weight), the drawn token (the same in
// the order of the index). Weights are added up per piece of the order's range in LDS, the few items of the piece that holds the target
// are ranked by a wave (sm_pick). It runs over a list in LDS of all tokens that may be kept, where that can hold them: what may
// be kept is known early, since where r of 1024 threads' own largest logits reach a value, at least r of the row do, and few
// more. Where it cannot, the row is cut into pieces of 1 / SM_FINE in (m - x) / t first, and the list holds one of them.
//
// What bounds it, at 256 rows of 150001 (fp32, a workgroup each; greedy rows, read once, 24.6 us, 6.2 TB/s): the row is gone over twice, its
// largest logit first. Top-k 50 and min-p 0.05 of a list take 50 and 47 us, two readings. A weight is 22 fp64 instructions (they issue as fast as
// fp32 ones: 1.8 ns a wave and SIMD, profiles/hw_probe_stream_and_issue.txt) among some 30 in all, so it is taken where it is needed only:
// for all tokens 69 us, of which vector instructions are 37; top-p 0.9 needs every weight too, for the sum, and its piece, an LDS
// atomic: 115 us, 62 of instructions. The list saves the passes that follow (a row of 32000 in one workgroup: 13 us for top-k, 27 for top-p);
// a nucleus of more than 8192 tokens costs them (temperature 1.5: 178 us).
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
#define SM_REST_P 3        // ... and top-p tries the tokens above all but these of them (6000)
#define SM_LOWEST 0x00800000u  // order of the lowest finite logit
// Few rows are shared by several workgroups each, up to 16, as long as there is a CU for each of them (two do not fit into its LDS) and
// the row is long: 1 row of 32000, in two, 17 to 18 us instead of 13 (top-k), 31 either way (top-p); of 128000 in 16: 21 either way
// (top-k), 47 instead of 82 (top-p), 22 instead of 40 (all tokens).
#define SM_SPLIT_WGS 256
#define SM_SPLIT_VOCAB 65536
#define SM_SLICES 16
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
// target(all the weight). All threads call; ends behind a wait, and may be called again at once.
template <typename TARGET, typename EACH>
__device__ __forceinline__ sm_bin sm_locate(sm_shared& S, TARGET target_of, EACH each) {
  static_assert(SM_BINS == 2 * SM_NT, "two bins a thread");
  each([&](uint32_t bin, uint64_t weight) { atomicAdd((unsigned long long*)&S.bins[bin], (unsigned long long)weight); });
  __syncthreads();
  if (threadIdx.x == 0) S.found_bin = -1;  // (behind this wait all have read the call before's; the scan's comes before the bin is found)
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
// Of items (order, index, a function that gives the weight) that `each` hands to its argument, from the largest order down, equal ones by index: the one at
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
      each([&](uint32_t order, int index, auto weight) __attribute__((always_inline)) {
        if (ties && order != same) return;
        const uint32_t o = ties ? ~(uint32_t)index : order;
        if (o >= lo && o <= hi) f(o, order, index, weight());
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

// A row: its settings, its largest logit, and the pieces of 1 / SM_FINE in (m - x) / t that it is cut into, the last one for all that is further down
template <int DT>
struct sm_row {
  static constexpr int ES = DT == SAH_F32 ? 4 : 2, E = 16 / ES;
  static constexpr int U = 4, SEG = SAH_WAVE * E * U;  // a segment: what a wave reads in U turns
  const void* x;
  int V, k;
  float temp, p, least;
  bool use_k, use_p, use_m;
  float best, fine;
  int best_at;
  __device__ __forceinline__ sm_row(const sah_sample_args& P, int r) {
    V = P.vocab;
    x = (const char*)P.logits + (int64_t)r * P.row_pitch * ES;
    temp = P.temperatures ? P.temperatures[r] : P.temperature;
    k = P.top_ks ? P.top_ks[r] : P.top_k;
    p = P.top_ps ? P.top_ps[r] : P.top_p;
    least = P.min_ps ? P.min_ps[r] : P.min_p;
    least = least > 1.f ? 1.f : least;
    use_k = k > 0 && k < V;
    use_p = p < 1.f;
    use_m = least > 0.f;
  }
  __device__ __forceinline__ void largest(float value, int at) {
    best = value;
    best_at = at;
    fine = SM_FINE / temp;
  }
  __device__ __forceinline__ bool one_answer() const { return best == -INFINITY || !(temp > 0.f); }
  __device__ __forceinline__ bool listed() const { return (use_k || use_p || use_m) && (V <= SM_CAP || !use_k || k <= SM_RANK_K); }
  __device__ __forceinline__ bool total() const { return use_p && !use_k && V > SM_CAP; }  // every weight is needed for top-p
  __device__ __forceinline__ bool everything() const { return !use_k && !use_p && !use_m; }
  __device__ __forceinline__ int piece(float v) const {
    const float d = (best - v) * fine;
    return v == best ? 0 : d < SM_BINS - 1 ? (int)d : SM_BINS - 1;
  }
  // orders that no token of the piece is below, or above (a hundredth of a piece is more than all roundings, and these are monotonic)
  __device__ __forceinline__ uint32_t piece_low(int at) const {
    const float v = best - ((float)at + 1.01f) / fine;
    return at < SM_BINS - 1 && v > -INFINITY && v < best ? sm_order(v) : SM_LOWEST;
  }
  __device__ __forceinline__ uint32_t piece_high(int at) const {
    const float v = best - ((float)at - 0.01f) / fine;
    return at > 0 && v > -INFINITY && v < best ? sm_order(v) : sm_order(best);
  }
  // whole numbers before a token are less than p times the sum where they are less than that rounded up; the first is kept
  __device__ __forceinline__ uint64_t nucleus(uint64_t all) const {
    const double limit = ceil((double)p * (double)all);
    return limit > 1.0 ? (uint64_t)limit : 1;
  }
};

struct sm_top { float value, low; int at; };
// Over the workgroup: the largest value and the first place of it, and the smallest value above -inf (all -inf: +inf).
__device__ __forceinline__ sm_top sm_largest(sm_shared& S, float best, int best_at) {
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  float low = best > -INFINITY ? best : INFINITY;
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
  return sm_top{best, low, best_at};
}

struct sm_from {
  float value;     // the list holds the tokens of at least this
  bool complete;   // it has every token that min-p keeps
};
// own: the largest logit of this thread's share of the row (-inf: it has none). All threads call.
template <int DT>
__device__ __forceinline__ sm_from sm_list_from(sm_shared& S, const sm_row<DT>& row, float own, float low) {
  sm_from f{-INFINITY, true};
  if (row.V <= SM_CAP) return f;
  const uint32_t top = sm_order(row.best);
  if (row.use_k || row.use_p) {
    const uint32_t range = top - sm_order(low);
    const int bits = range ? 32 - __builtin_clz(range) : 0, shift = bits > 11 ? bits - 11 : 0;
    const sm_bin b = sm_locate(
        S, [&](uint64_t all) -> uint64_t { return row.use_k ? (uint64_t)row.k : all > SM_REST_P ? all - SM_REST_P : 1; },
        [&](auto put) { if (own > -INFINITY) put((top - sm_order(own)) >> shift, 1); });
    if (b.at >= 0) {
      const uint32_t down = ((uint32_t)(b.at + 1) << shift) - 1;  // to the lower end of the piece
      f.value = sm_value(down < range ? top - down : top - range);
      f.complete = false;
    }
  }
  if (row.use_m && !row.use_k) {
    // e >= least where x >= m + t ln(least); a little below that, for the roundings
    const sm_weights weigh(row.best, row.temp);
    const double at = weigh.m + (double)row.temp * log((double)row.least);
    const float below = (float)(at - 1e-6 * (fabs(at) + fabs(weigh.m)) - 1e-30);
    if (below > f.value || !row.use_p) {
      f.value = below == below ? below : -INFINITY;
      f.complete = true;
    }
  }
  return f;
}

__device__ __forceinline__ void sm_enlist(sm_shared& S, float v, int i) {
  const int n = atomicAdd(&S.count, 1);
  if (n < SM_CAP) S.list[n] = make_uint2(sah_float_to_bits(v), (uint32_t)i);
}
__device__ __forceinline__ void sm_begin(sm_shared& S) {
  for (int b = threadIdx.x; b < SM_BINS; b += SM_NT) S.bins[b] = 0;
  if (threadIdx.x == 0) S.count = S.n_small[0] = S.n_small[1] = 0;
}

// ---------------------------------------------------------------------------
// Few rows: the passes over a whole row are shared by up to SM_SLICES workgroups, in two kernels ahead of the row's own.
// ---------------------------------------------------------------------------
struct sm_work {  // of a row
  uint64_t bins[SM_BINS];    // weight of the pieces
  uint64_t segs[SM_NT];      // weight of the segments
  uint2 list[SM_CAP];
  float own[SM_NT];          // the largest logits of SM_NT shares of the row, -inf where a share is empty
  float best[SM_SLICES];     // ... of the slices
  int best_at[SM_SLICES];
  sm_from from;
  int count, count_again;
};

template <int DT>
struct sm_slice {
  int begin, n;  // tokens; n may be 0
  __device__ __forceinline__ sm_slice(int V, int number, int slices) {
    constexpr int SEG = sm_row<DT>::SEG;
    const int segs = (V + SEG - 1) / SEG, each = (segs + slices - 1) / slices * SEG;
    begin = number * each;  // (below 2^20 + 16 SEG)
    n = begin < V ? (V - begin < each ? V - begin : each) : 0;
  }
};

// Every slice's largest logit, and those of SM_NT / slices shares of it (slices: a power of two)
template <int DT>
__global__ __launch_bounds__(SM_NT, 4) void k_sample_largest(sah_sample_args P) {
  __shared__ float s_own[SM_NT];
  SAH_DYNAMIC_LDS(s_dyn);
  sm_shared& S = *(sm_shared*)s_dyn;
  const sm_row<DT> row(P, blockIdx.y);
  const sm_slice<DT> slice(row.V, blockIdx.x, gridDim.x);
  sm_work& W = ((sm_work*)P.work)[blockIdx.y];
  const int bins = SM_BINS / (int)gridDim.x, shares = SM_NT / (int)gridDim.x;
  for (int b = threadIdx.x; b < bins; b += SM_NT) W.bins[blockIdx.x * bins + b] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) W.count = W.count_again = 0;
  float best = -INFINITY;
  int best_at = INT32_MAX;
  sm_each<DT, 4>((const char*)row.x + (int64_t)slice.begin * row.ES, slice.n, [&](float v, int i) {
    best_at = v > best ? i + slice.begin : best_at;
    best = v > best ? v : best;
  });
  s_own[threadIdx.x] = best;
  const sm_top top = sm_largest(S, best, best_at);  // (waits)
  if ((int)threadIdx.x < shares) {
    float own = -INFINITY;
    for (int t = threadIdx.x; t < SM_NT; t += shares) own = fmaxf(own, s_own[t]);
    W.own[blockIdx.x * shares + threadIdx.x] = own;
  }
  if (threadIdx.x == 0) {
    W.best[blockIdx.x] = top.value;
    W.best_at[blockIdx.x] = top.at;
  }
}

// the row's largest logit out of its slices'
template <int DT>
__device__ __forceinline__ void sm_largest_of(sm_row<DT>& row, const sm_work& W, int slices) {
  float best = -INFINITY;
  int at = INT32_MAX;
  for (int i = 0; i < slices; ++i) {  // in the order of the index
    at = W.best[i] > best ? W.best_at[i] : at;
    best = fmaxf(best, W.best[i]);
  }
  row.largest(best, at);
}

// Writes the weights of the segments of [begin, begin + n), a wave's turn each. plain: weight is sm_fixed(weigh(v)).
template <int DT, typename WEIGHT>
__device__ __forceinline__ void sm_segments(const sm_row<DT>& row, int begin, int n, bool plain, const sm_weights& weigh, uint64_t* segs, WEIGHT weight) {
  constexpr int ES = sm_row<DT>::ES, E = sm_row<DT>::E, U = sm_row<DT>::U, SEG = sm_row<DT>::SEG;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id(), end = begin + n;
  const int n_segs = (n + SEG - 1) / SEG;
  auto place = [&](int j) { return begin + (wave + j / U * SM_NW) * SEG + (j % U * SAH_WAVE + lane) * E; };  // this lane's j-th piece
  auto load = [&](int i) __attribute__((always_inline)) -> sah_u4 { return i + E <= end ? *(const sm_vec*)((const char*)row.x + (int64_t)i * ES) : sah_u4{0, 0, 0, 0}; };
  sah_u4 next = load(place(0));
  uint64_t part = 0;
#pragma unroll 1
  for (int j = 0; wave + j / U * SM_NW < n_segs; ++j) {
    const sah_u4 v = next;
    const int i = place(j);
    next = load(place(j + 1));
    if (i + E <= end && plain) {
#pragma unroll
      for (int e = 0; e < E; ++e) part += sm_raw(weigh(sm_unpack<DT>(v, e)));
      part -= E * SM_ZERO;
    } else if (i + E <= end) {
#pragma unroll
      for (int e = 0; e < E; ++e) part += weight(sm_unpack<DT>(v, e), i + e);
    } else {
#pragma unroll 1
      for (int e = 0; i + e < end; ++e) part += weight(sah_load<DT>(row.x, i + e), i + e);
    }
    if (j % U == U - 1) {
      part = sah_lane_u64(sah_wave_incl_scan_u64(part), SAH_WAVE - 1);
      if (lane == 0) segs[begin / SEG + wave + j / U * SM_NW] = part;
      part = 0;
    }
  }
}

// The slice's list to the row's; where that cannot hold all slices', `count` says so. All threads call, behind a wait.
__device__ __forceinline__ void sm_hand_over(sm_shared& S, sm_work& W, int& count) {
  const int n = S.count;
  if (threadIdx.x == 0) S.found_bin = atomicAdd(&count, n);
  __syncthreads();
  const int at = S.found_bin;
  if (n > SM_CAP || at > SM_CAP - n) return;
  for (int j = threadIdx.x; j < n; j += SM_NT) W.list[at + j] = S.list[j];
}
// ... and from there, all requested at once; more than SM_CAP: nothing
__device__ __forceinline__ void sm_take_list(sm_shared& S, const sm_work& W, int n) {
  constexpr int N = SM_CAP / (2 * SM_NT);
  if (n > SM_CAP) return;
  sah_u4 two[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = 2 * ((int)threadIdx.x + i * SM_NT);
    if (j < n) two[i] = *(const sah_u4*)&W.list[j];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = 2 * ((int)threadIdx.x + i * SM_NT);
    if (j < n) *(sah_u4*)&S.list[j] = two[i];
  }
}
// top-p's last token: the weight that it reaches, and its piece. (The bins are LDS's own again afterwards.)
template <int DT>
__device__ __forceinline__ sm_bin sm_border(sm_shared& S, const sm_row<DT>& row, const sm_work& W, uint64_t& whole) {
  return sm_locate(S, [&](uint64_t all) { return whole = row.nucleus(all); },
                   [&](auto) { *(sah_u4*)&S.bins[2 * threadIdx.x] = *(const sah_u4*)&W.bins[2 * threadIdx.x]; });
}
template <int DT>
__device__ __forceinline__ bool sm_too_short(const sm_row<DT>& row, const sm_from& from, const sm_bin& border) {
  return from.value > -INFINITY && !from.complete && row.piece(from.value) <= border.at;
}

// Every slice's tokens for the list, and the weights of its pieces or segments
template <int DT>
__global__ __launch_bounds__(SM_NT, 4) void k_sample_slices(sah_sample_args P) {
  SAH_DYNAMIC_LDS(s_dyn);
  sm_shared& S = *(sm_shared*)s_dyn;
  sm_row<DT> row(P, blockIdx.y);
  const sm_slice<DT> slice(row.V, blockIdx.x, gridDim.x);
  sm_work& W = ((sm_work*)P.work)[blockIdx.y];
  sm_largest_of(row, W, gridDim.x);
  if (row.one_answer()) return;
  const sm_weights weigh(row.best, row.temp);
  if (row.everything()) {
    sm_segments<DT>(row, slice.begin, slice.n, true, weigh, W.segs, [&](float v, int) { return sm_fixed(weigh(v)); });
    return;
  }
  if (!row.listed()) return;
  sm_begin(S);
  const float own = W.own[threadIdx.x];
  const sm_top top = sm_largest(S, own, 0);  // (waits)
  const sm_from from = sm_list_from<DT>(S, row, own, top.low);
  if (blockIdx.x == 0 && threadIdx.x == 0) W.from = from;
  const void* x = (const char*)row.x + (int64_t)slice.begin * row.ES;
  auto enlist = [&](float v, int i) __attribute__((always_inline)) { if (v >= from.value && v > -INFINITY) sm_enlist(S, v, i + slice.begin); };
  if (row.total()) {
    sm_each<DT, 1>(x, slice.n, [&](float v, int i) {
      enlist(v, i);
      atomicAdd((unsigned long long*)&S.bins[row.piece(v)], (unsigned long long)sm_fixed(weigh(v)));
    });
  } else {
    sm_each<DT, 4>(x, slice.n, enlist);
  }
  __syncthreads();
  if (row.total())
    for (int b = threadIdx.x; b < SM_BINS; b += SM_NT)
      if (S.bins[b]) atomicAdd((unsigned long long*)&W.bins[b], (unsigned long long)S.bins[b]);
  sm_hand_over(S, W, W.count);
}

// Rows whose top-p reaches further down than their list: the list anew, all down to there
template <int DT>
__global__ __launch_bounds__(SM_NT, 4) void k_sample_list(sah_sample_args P) {
  SAH_DYNAMIC_LDS(s_dyn);
  sm_shared& S = *(sm_shared*)s_dyn;
  sm_row<DT> row(P, blockIdx.y);
  if (!row.total()) return;
  sm_work& W = ((sm_work*)P.work)[blockIdx.y];
  sm_largest_of(row, W, gridDim.x);
  if (row.one_answer()) return;
  uint64_t whole;
  const sm_bin border = sm_border(S, row, W, whole);
  if (!sm_too_short(row, W.from, border)) return;
  if (threadIdx.x == 0) S.count = 0;
  __syncthreads();
  const sm_slice<DT> slice(row.V, blockIdx.x, gridDim.x);
  sm_each<DT, 4>((const char*)row.x + (int64_t)slice.begin * row.ES, slice.n, [&](float v, int i) __attribute__((always_inline)) {
    if (v > -INFINITY && row.piece(v) <= border.at) sm_enlist(S, v, i + slice.begin);
  });
  __syncthreads();
  sm_hand_over(S, W, W.count_again);
}

// SPLIT: by `slices` workgroups' work so far
template <int DT, bool SPLIT>
__global__ __launch_bounds__(SM_NT, 4) void k_sample(sah_sample_args P, int slices) {
  sah_touch_kernargs<sizeof(sah_sample_args)>();
  SAH_DYNAMIC_LDS(s_dyn);
  sm_shared& S = *(sm_shared*)s_dyn;
  constexpr int E = sm_row<DT>::E, U = sm_row<DT>::U, SEG = sm_row<DT>::SEG;
  const int r = blockIdx.x;
  sm_row<DT> row(P, r);
  const int V = row.V, k = row.k;
  const void* x = row.x;
  const float least = row.least;
  const bool use_k = row.use_k, use_p = row.use_p, use_m = row.use_m;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  [[maybe_unused]] const sm_work& W = ((const sm_work*)P.work)[SPLIT ? r : 0];
  sm_begin(S);
  int round = 0;

  // the largest logit and its first place
  [[maybe_unused]] float own = -INFINITY, low = INFINITY;
  if constexpr (SPLIT) {
    sm_largest_of(row, W, slices);
    __syncthreads();
  } else {
    int own_at = INT32_MAX;
    sm_each<DT, 4>(x, V, [&](float v, int i) {
      own_at = v > own ? i : own_at;
      own = v > own ? v : own;
    });
    const sm_top top = sm_largest(S, own, own_at);
    low = top.low;
    row.largest(top.value, top.at);
  }
  const float best = row.best;
  if (row.one_answer()) {
    if (threadIdx.x == 0) {
      P.tokens[r] = best == -INFINITY ? -1 : row.best_at;
      if (P.logprobs) P.logprobs[r] = best == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const sm_weights weigh(best, row.temp);
  const uint32_t top = sm_order(best);
  auto piece = [&](float v) { return row.piece(v); };
  auto nucleus = [&](uint64_t all) { return row.nucleus(all); };
  // kept: logits above thr, and of those equal to it the ones with an index up to last
  float thr = -INFINITY;
  int last = -1;
  auto kept = [&](float v, int i) { return v > thr || (v == thr && i <= last); };
  int n_list = 0;
  auto list_again = [&](auto take) __attribute__((always_inline)) {  // a new list, of the kept tokens that `take` takes; whether it holds them
    if (threadIdx.x == 0) S.count = 0;
    __syncthreads();
    sm_each<DT, 1>(x, V, [&](float v, int i) { if (kept(v, i) && take(v)) sm_enlist(S, v, i); });
    __syncthreads();
    n_list = S.count;
    return n_list <= SM_CAP;
  };

  // the tokens that may be kept, in a list, where they are not too many
  bool list = false;
  const bool total = row.total();
  uint64_t whole = 0;                  // total: the weight that top-p's last token reaches ...
  sm_bin border{0, 0};                 // ... and its piece
  uint32_t lowest = SM_LOWEST;         // no token of the list is of a lower order
  if (row.listed()) {
    sm_from from;
    if constexpr (SPLIT) {
      from = W.from;
      n_list = W.count;
      if (!total) sm_take_list(S, W, n_list);
    } else {
      from = sm_list_from<DT>(S, row, own, low);
    }
    if (from.value > -INFINITY && from.value < best) lowest = sm_order(from.value);
    if (total) {
      // the weights' pass shares the row out into pieces too: if top-p's last token lies below the list, its piece is known
      if constexpr (SPLIT) {
        border = sm_border(S, row, W, whole);
      } else {
        border = sm_locate(
            S, [&](uint64_t all) { return whole = nucleus(all); },
            [&](auto put) __attribute__((always_inline)) {
              sm_each<DT, 1>(x, V, [&](float v, int i) {
                if (v >= from.value && v > -INFINITY) sm_enlist(S, v, i);
                put(piece(v), sm_fixed(weigh(v)));
              });
            });
        n_list = S.count;
      }
      if (sm_too_short(row, from, border)) {
        // all down to there, if the list holds that
        if constexpr (SPLIT) {
          n_list = W.count_again;
        } else {
          list_again([&](float v) { return piece(v) <= border.at; });
        }
      }
      if constexpr (SPLIT) sm_take_list(S, W, n_list);
    } else if constexpr (!SPLIT) {
      sm_each<DT, 4>(x, V, [&](float v, int i) { if (v >= from.value && v > -INFINITY) sm_enlist(S, v, i); });
      __syncthreads();
      n_list = S.count;
    }
    __syncthreads();
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
    auto target_of = [&](uint64_t all) -> uint64_t { return !stage ? k : total ? whole - border.before : nucleus(all); };
    auto items = [&](bool from_list) {
      return [&, from_list](auto put) __attribute__((always_inline)) {
        // (top-p's last token lies in the border's piece)
        each(from_list, [&](float v, int i) __attribute__((always_inline)) {
          if (kept(v, i) && (!total || piece(v) == border.at)) put(sm_order(v), i, [&] { return weight(v); });
        });
      };
    };
    sm_item found{false, 0, 0};
    if (list) {
      found = sm_pick(S, round, total ? row.piece_low(border.at) : lowest, total ? row.piece_high(border.at) : top, target_of, items(true));
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
        found = sm_pick(S, round, row.piece_low(b.at), row.piece_high(b.at), rest, items(true));
      } else {  // (thousands of logits in one piece)
        found = sm_pick(S, round, row.piece_low(b.at), row.piece_high(b.at), rest, [&](auto put) __attribute__((always_inline)) {
          each(false, [&](float v, int i) { if (kept(v, i) && piece(v) == b.at) put(sm_order(v), i, [&] { return weight(v); }); });
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
        [&](auto put) __attribute__((always_inline)) { each(true, [&](float v, int i) { put(~(uint32_t)i, i, [&] { return final_weight(v, i); }); }); });
    if (threadIdx.x == 0) answer(f.index, all);
    return;
  }
  // The whole row: the weights of its segments; then inside the one that holds the target.
  static_assert(SM_MAX_VOCAB / SEG <= SM_NT && SM_NT <= SM_CAP, "a sum a thread");
  const int n_segs = (V + SEG - 1) / SEG;
  const uint64_t* segs = (const uint64_t*)S.list;
  if (SPLIT && row.everything()) {
    segs = W.segs;
  } else {
    __syncthreads();  // the list is no longer read
    sm_segments<DT>(row, 0, V, thr == -INFINITY && !use_m, weigh, (uint64_t*)S.list, final_weight);
    __syncthreads();
  }
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
// Workgroups a row (a power of two)
static int sm_slices(const sah_sample_args* a) {
  if (a->n_rows <= 0 || a->vocab < SM_SPLIT_VOCAB || (!a->temperatures && !(a->temperature > 0.f))) return 1;  // (one pass is all that is done)
  int n = 1;
  while (n < SM_SLICES && 2 * n * (int64_t)a->n_rows <= SM_SPLIT_WGS) n *= 2;
  return n;
}
extern "C" int64_t sah_sample_work_bytes(const sah_sample_args* a) {
  return a && sm_slices(a) > 1 ? (int64_t)a->n_rows * (int64_t)sizeof(sm_work) : 0;
}

template <int DT>
static int sm_launch(const sah_sample_args* a, int slices) {
  hipStream_t st = (hipStream_t)a->stream;
  auto kernel = slices > 1 ? k_sample<DT, true> : k_sample<DT, false>;
  if (int rc = sah_allow_lds((const void*)kernel, sizeof(sm_shared), "sah_sample_tokens")) return rc;
  if (slices > 1) {
    if (int rc = sah_allow_lds((const void*)k_sample_largest<DT>, sizeof(sm_shared), "sah_sample_tokens")) return rc;
    if (int rc = sah_allow_lds((const void*)k_sample_slices<DT>, sizeof(sm_shared), "sah_sample_tokens")) return rc;
    {
      sah_timed timed("k_sample_largest", a->stream);
      hipLaunchKernelGGL(k_sample_largest<DT>, dim3(slices, a->n_rows), dim3(SM_NT), sizeof(sm_shared), st, *a);
      if (int rc = sah_launch_status("sah_sample_tokens(largest)")) return rc;
    }
    {
      sah_timed timed("k_sample_slices", a->stream);
      hipLaunchKernelGGL(k_sample_slices<DT>, dim3(slices, a->n_rows), dim3(SM_NT), sizeof(sm_shared), st, *a);
      if (int rc = sah_launch_status("sah_sample_tokens(slices)")) return rc;
    }
    if ((a->top_ps || a->top_p < 1.f) && (a->top_ks || a->top_k <= 0 || a->top_k >= a->vocab)) {  // (some row may go by all its weights)
      if (int rc = sah_allow_lds((const void*)k_sample_list<DT>, sizeof(sm_shared), "sah_sample_tokens")) return rc;
      sah_timed timed("k_sample_list", a->stream);
      hipLaunchKernelGGL(k_sample_list<DT>, dim3(slices, a->n_rows), dim3(SM_NT), sizeof(sm_shared), st, *a);
      if (int rc = sah_launch_status("sah_sample_tokens(list)")) return rc;
    }
  }
  sah_timed timed("k_sample", a->stream);
  hipLaunchKernelGGL(kernel, dim3(a->n_rows), dim3(SM_NT), sizeof(sm_shared), st, *a, slices);
  return sah_launch_status("sah_sample_tokens");
}

extern "C" int sah_sample_tokens(const sah_sample_args* a) {
  if (!a) return sah_fail(SAH_ENULL, "sah_sample_tokens: args is NULL");
  if (a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16) return sah_fail(SAH_EDTYPE, "sah_sample_tokens: dtype %d", a->dtype);
  if (a->n_rows < 0 || a->vocab <= 0) return sah_fail(SAH_EINVAL, "sah_sample_tokens: n_rows must be >= 0, vocab > 0");
  if (a->vocab > SM_MAX_VOCAB) return sah_fail(SAH_ESHAPE, "sah_sample_tokens: vocab %d; at most %d", a->vocab, SM_MAX_VOCAB);
  if (a->row_pitch < a->vocab && a->n_rows > 1) return sah_fail(SAH_EINVAL, "sah_sample_tokens: row_pitch is less than vocab");
  if (a->n_rows == 0) return SAH_OK;
  if (!a->logits || !a->uniforms || !a->tokens) return sah_fail(SAH_ENULL, "sah_sample_tokens: NULL pointer");
  const int64_t need = sah_sample_work_bytes(a);
  if (a->work && ((uint64_t)a->work % 16 || a->work_bytes < need)) return sah_fail(SAH_ECAPACITY, "sah_sample_tokens: work is too small, or not on a multiple of 16 bytes");
  const int slices = a->work && need ? sm_slices(a) : 1;
  if (a->dtype == SAH_F32) return sm_launch<SAH_F32>(a, slices);
  return a->dtype == SAH_BF16 ? sm_launch<SAH_BF16>(a, slices) : sm_launch<SAH_F16>(a, slices);
}
