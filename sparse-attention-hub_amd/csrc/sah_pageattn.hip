// Attention over pages in 8 bits, or over the pages that a list names for each token: few rows a request, so that reading keys and values bounds it
// (64 answers of 1K to 32K 8-bit keys, 8 key heads of 128: 2.2 GB in 384 us, 5.8 TB/s), and where a call is small the time of a workgroup's chain of
// reads: lengths, table, keys, values (one answer over 1024 listed keys: 11 us, 7 of them before the first product).
//
// Of a request's tokens (with a list: of one token) and a key head's query heads every (token, head) is a row; up to 16 are a tile. All
// tiles of all requests are one line of work, measured in keys; every workgroup takes an equal piece of it, whatever the requests' lengths (where there is
// little work, a piece of one tile), finds its place from the lengths on the device, and works through tiles and parts of tiles. A part's (m, l, acc) goes to the workspace, a second
// kernel joins the parts of a row.
//
// The four waves of a workgroup take 32 keys of a tile in turn. Nothing is staged: keys and values
// go from memory to the registers in which the matrix instructions want them. S^T = K Q^T (16 keys x 16 rows a tile of the matrix): a lane reads 16
// bytes of a key's row, the 4 lanes of a key 64 neighbouring ones. The result has row n in lanes n + 16 g, keys 4 g .. 4 g + 3 of both key
// tiles, which is what O^T = V^T P^T wants of P with its key slots in that order; of V lane i + 16 g then holds the 8 keys' dims
// C i .. C i + C - 1 (a key's row is 16 lanes' pieces, one after the other), and a permutation of 16-bit halves inside the lane makes of
// them the operand of dim C i + e, the output's tile e. 8-bit elements become bf16 on the way, their scale with them, in one instruction a pair: exact.
// A 32-key step's K is requested as soon as the step before has been multiplied with its own, V likewise: half a step or more is under way at all times.
// (Two steps ahead: 412 instead of 404 us, lists that several tokens share 85 instead of 59: the registers cost waves.)
#include "sah_pages.h"

#define PT_NT 256
#define PT_NW (PT_NT / SAH_WAVE)
#define PT_ROWS 16
#define PT_STEP 32                      // keys of a wave's step
#define PT_MOST 2048                    // keys whose pages a workgroup looks up at once
#define PT_CUS 256
#define PT_XCDS 8
#define PT_LAST_CACHE 0x1p28               // bytes
// What starting and ending a tile takes, in keys: how pieces with many tiles are balanced against those with one (256 and 384: within 2 us of 400).
#define PT_TILE_COST 128
// Keys a workgroup below which every tile is cut by itself (16 answers of 1K to 2K keys 29.9 -> 24.9 us, drafts within a window 24.1 -> 19.6; what decides
// it costs other calls 0.6 us). Beyond, the balance of equal pieces is worth more (8 answers of 8192 keys, 520 a workgroup: 36.4 us against 39.3).
#define PT_FEW 512
// The least that is worth a workgroup, in keys of one byte an element: wider ones are worth one sooner. (272 listed fp32 keys a token, 2 key heads: pieces
// of 64 keys 18 us, of 256 23; 8-bit drafts within a window: of 256 keys 27 us, of 64 30.)
#define PT_LEAST 256

struct pt_args {
  sah_page_attention_args a;
  int tokens, blocks;     // tokens of a tile; tiles that a token's query heads of a key head make
  int unit;               // window: keys that begin and end with one
  int least;              // keys of a key head that are worth a workgroup
  // Key heads that a workgroup works on at once, each by as many of its waves: 4, 2 or 1. Their keys lie side by side, which memory rewards (64
  // answers of 1K to 32K keys, 8 heads: 445 us one by one, 407 by 4; 32 of 4K to 8K: 106 by 1, 97 by 2, 94 by 4); the fewer, the fewer parts
  // there are to join (one answer of 32K keys: 32.1 us by 4, 27.6 by 2, 26.7 by 1; of 128K: 70.5, 66.8, 71.9). With a list each has pages of its own, and 1 it is.
  int heads;
  int n_lost;             // the call that stands in for one over a copy: bytes that tell whether it has to
  const uint8_t* lost;
};

template <int KT, int QT>
struct pt_types {
  static constexpr int MT = KT == SAH_E4M3 ? SAH_BF16 : KT;     // what is multiplied
  // Terms of MT's bits that a query and a weight are taken apart into: a query has all of its bits, a weight 16 or more (fp32: 24).
  static constexpr int NQ = KT != SAH_E4M3 || QT == SAH_BF16 ? 1 : QT == SAH_F16 ? 2 : 3;
  static constexpr int NP = KT == SAH_F32 ? 1 : KT == SAH_E4M3 && QT == SAH_F32 ? 3 : 2;
  // How far a row's maximum may rise, in powers of two, before the row is rescaled; and the power of two that weights are held above their
  // size by, for fp16 terms of weights far below the largest.
  static constexpr float SLACK = MT == SAH_F16 ? 6.0f : 8.0f;
  static constexpr float SCALE = MT == SAH_F16 ? 8.0f : 0.0f;
};

// The kernel's arguments where they lie. Each call gives an address that the compiler knows nothing of, so that what is read behind it is read again
// for every tile, instead of being kept in scalar registers, of which there are too few.
typedef const pt_args __attribute__((address_space(4))) pt_karg;
__device__ __forceinline__ const pt_args& pt_arguments() {
#if defined(__HIP_DEVICE_COMPILE__)
  pt_karg* p = (pt_karg*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const pt_args*)p;
#else
  static pt_args* none;
  return *none;
#endif
}

// From products to powers of two. The sign is the query's; 0 is a number so small that all weights are 1.
__device__ __forceinline__ float pt_log2(float scaling) { return fmaxf(fabsf(scaling) * 1.4426950408889634f, 1e-37f); }

// Keys by number: u = 0, 1, ... are the keys that some row of the tile may see, in the order of the cache (a list: of the list).
struct pt_keys {
  int n;          // of them
  int hi;         // the last key that a row sees, or -1
  int sinks;      // window: the first ones, a multiple of `unit`
  int skip;       // ... what lies between them and the others
};
__device__ __forceinline__ pt_keys pt_keys_of(const pt_args& A, const pg_request& r, int64_t p_lo, int64_t p_hi) {
  const sah_page_attention_args& P = A.a;
  pt_keys k{0, -1, 0, 0};
  if (p_hi < 0 || r.kv == 0) return k;
  k.hi = p_hi < r.kv ? (int)p_hi : r.kv - 1;
  if (P.pages) {
    k.n = P.n_select * P.cache.page_size;  // (the host has checked that it fits)
    return k;
  }
  k.n = k.hi + 1;
  if (P.window) {
    const int64_t first = p_lo - P.window + 1;
    const int from = first > 0 ? (int)(first < k.hi + 1 ? first : k.hi + 1) / A.unit * A.unit : 0;
    const int sink = P.sink < k.hi + 1 ? P.sink : k.hi + 1;
    const int64_t sinks = ((int64_t)sink + A.unit - 1) / A.unit * A.unit;
    if (sinks < from) {
      k.sinks = (int)sinks;
      k.skip = from - k.sinks;
      k.n -= k.skip;
    }
  }
  return k;
}

// ---------------------------------------------------------------------------
// where the work is
// ---------------------------------------------------------------------------
// Cost of a request's tiles, all of them alike: about the keys that its last tile reads. Only the balance depends on it.
struct pt_cost {
  int64_t each;
  int64_t tiles;  // of all groups of key heads
  __device__ __forceinline__ int64_t all() const { return each * tiles; }
};
struct pt_lens { int begin, end, kv; };
__device__ __forceinline__ pt_lens pt_lens_of(const sah_page_requests& R, int b) { return pt_lens{R.cu_new[b], R.cu_new[b + 1], R.kv_lens[b]}; }
__device__ __forceinline__ pt_cost pt_cost_of(const pt_args& A, const pt_lens& lens) {
  const sah_page_attention_args& P = A.a;
  const sah_page_requests& R = P.requests;
  const int begin = lens.begin, end = lens.end, kv = lens.kv;
  pt_cost c{PT_TILE_COST, 0};
  const int last = end < R.n_tokens ? end : R.n_tokens;
  if (begin < 0 || begin >= last) return c;
  c.tiles = (int64_t)((last - begin + A.tokens - 1) / A.tokens) * A.blocks * (P.cache.Hkv / A.heads);
  int64_t n = (int64_t)kv - end + last;  // keys up to the last row's position
  const int64_t most = (int64_t)R.table_width * P.cache.page_size;
  if (P.pages) {
    n = (int64_t)P.n_select * P.cache.page_size;  // (the same for all tiles: pt_start counts on it)
  } else {
    n = n < most ? n : most;
    if (P.window && (int64_t)P.sink + P.window + 2 * (int64_t)A.unit < n) n = (int64_t)P.sink + P.window + 2 * (int64_t)A.unit;
  }
  c.each += n > 0 ? n : 0;
  return c;
}
// How the line is shared: by `n` workgroups, and where workgroup w's piece begins
struct pt_shares {
  int64_t each;
  uint32_t n, rest;
  int w0, parts;  // parts > 0: the piece is one of so many of a tile, the first of them workgroup w0's
  __device__ __forceinline__ int64_t bound(int w) const { return each * w + rest * (uint32_t)w / n; }  // (n is at most 1024)
  // Whose piece has key x, `away` from where w's begins: asked for two keys at once, by the halves of a wave, whose lanes try a piece each. (The
  // guess is off by one at most: pieces differ by one key.)
  __device__ __forceinline__ void holders(int64_t x, int64_t away, int w, int& lower, int& upper) const {
    const int lane = threadIdx.x & (SAH_WAVE - 1), guess = w - 16 + (int)floorf((float)away / ((float)each + (float)rest / (float)n)), c = guess + (lane & 31);
    const uint64_t begun = __ballot((c >= 0) & (c < (int)n) & (bound(c) <= x));
    lower = __builtin_amdgcn_readlane(guess, 0) + 31 - __builtin_clz((uint32_t)begun | 1u);
    upper = __builtin_amdgcn_readlane(guess, 32) + 31 - __builtin_clz((uint32_t)(begun >> 32) | 1u);
  }
};
__device__ __forceinline__ pt_shares pt_share(const pt_args& A, int64_t total, int wgs) {
  pt_shares s;
  const int64_t w = (total * A.heads + A.least - 1) / A.least;
  s.n = (uint32_t)(w < wgs ? w : wgs);
  s.each = s.n ? pg_uniform(pg_div(total, s.n)) : 0;
  s.rest = (uint32_t)(total - s.each * s.n);
  s.w0 = s.parts = 0;
  return s;
}
// Neighbours on the line share keys' cache lines (scales, and what lies between two heads), so they get the same XCD.
__device__ __forceinline__ int pt_number() { return (int)(blockIdx.x % PT_XCDS) * (int)(gridDim.x / PT_XCDS) + (int)(blockIdx.x / PT_XCDS); }

// A place on the line: request, tile of it, where the tile begins
struct pt_place {
  int b;
  pt_lens lens;
  int64_t tile, begin;
  pt_cost cost;
  int64_t x0, x1;  // the workgroup's piece
};
// Cost of a piece where no piece holds parts of two tiles, or 0 where pieces are equal. A second tile costs a workgroup as much as its first one's start, some 7
// us, so calls of little work a workgroup cut every tile by itself, and those whose tiles are alike or few do, which lose no balance by it. At most
// `wgs` pieces: total / target + tiles.
__device__ __forceinline__ int64_t pt_target(const pt_args& A, int64_t total, int64_t tiles, int wgs) {
  if (tiles == 0 || tiles > wgs) return 0;
  const int64_t least = A.least / A.heads, room = wgs - tiles, target = room ? pg_uniform(pg_div(total + room - 1, room)) : total;
  if (!A.a.pages && A.a.requests.n_requests > 1 && tiles * 16 >= wgs && target > PT_FEW) return 0;
  return target > least ? target : least;
}
// s_sum: 2 PT_NW + 3 words; s_shares: how the line is shared. All threads call. False: no piece.
__device__ __forceinline__ bool pt_start(const pt_args& A, int w, int wgs, int64_t* s_sum, pt_shares& s_shares, pt_place& at) {
  const sah_page_requests& R = A.a.requests;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  // inclusive sum of v, and the sums of v and u over all threads
  auto scan = [&](int64_t v, int64_t u, int64_t& all, int64_t& all_u) -> int64_t {
    const int64_t incl = (int64_t)sah_wave_incl_scan_u64((uint64_t)v), incl_u = (int64_t)sah_wave_incl_scan_u64((uint64_t)u);
    __syncthreads();
    if (lane == SAH_WAVE - 1) {
      s_sum[wave] = incl;
      s_sum[PT_NW + wave] = incl_u;
    }
    __syncthreads();
    int64_t before = 0;
    all = all_u = 0;
#pragma unroll
    for (int i = 0; i < PT_NW; ++i) {
      before += i < wave ? s_sum[i] : 0;
      all += s_sum[i];
      all_u += s_sum[PT_NW + i];
    }
    all = pg_uniform(all);
    all_u = pg_uniform(all_u);
    return before + incl;
  };
  pt_lens lens{0, 0, 0};
  auto cost_of = [&](int b) -> pt_cost {
    if (b >= R.n_requests) return pt_cost{PT_TILE_COST, 0};
    lens = pt_lens_of(R, b);
    return pt_cost_of(A, lens);
  };
  // requests' costs and tiles, then where each one's pieces begin (of a line in keys, or in pieces), PT_NT requests at a time
  int64_t total = 0, tiles = 0, unused;
  pt_cost c{PT_TILE_COST, 0};
  for (int b = threadIdx.x; b < R.n_requests; b += PT_NT) {
    c = cost_of(b);
    total += c.all();
    tiles += c.tiles;
  }
  if (threadIdx.x == 0) s_sum[2 * PT_NW] = -1;
  const int64_t end_0 = scan(total, tiles, total, tiles);
  const int64_t target = pt_target(A, total, tiles, wgs);
  at.x0 = w;
  if (!target) {
    const pt_shares shares = pt_share(A, total, wgs);
    if (w >= (int)shares.n) return false;
    at.x0 = shares.bound(w);
    at.x1 = shares.bound(w + 1);
    if (threadIdx.x == 0) s_shares = shares;
  }
  int64_t run = 0;
  const bool alike = (A.a.pages || R.n_requests == 1) && tiles > 0;
  const int64_t each = alike ? pg_uniform(pg_div(total, tiles)) : 0;
  for (int b0 = 0; b0 < R.n_requests; b0 += PT_NT) {
    const int b = b0 + (int)threadIdx.x;
    if (R.n_requests > PT_NT) c = cost_of(b);
    const int64_t k = target ? pg_div((alike ? each : c.each) + target - 1, target) : 1, mine = target ? c.tiles * k : c.all();
    int64_t all = 0, end = end_0;
    if (R.n_requests > PT_NT || (target && !alike)) {
      end = run + scan(mine, 0, all, unused);
    } else if (target) {  // tiles of one cost: the first scan tells them, too
      end = pg_div(end_0, each) * k;
      all = tiles * pg_uniform(k);
    }
    if (mine && end > at.x0 && end - mine <= at.x0) {  // one thread's request holds x0
      s_sum[2 * PT_NW] = (int64_t)lens.kv << 32 | (uint32_t)b;
      s_sum[2 * PT_NW + 1] = end - mine;
      s_sum[2 * PT_NW + 2] = (int64_t)lens.end << 32 | (uint32_t)lens.begin;
    }
    run += all;
  }
  if (target && w >= run) return false;
  __syncthreads();
  const int64_t own = pg_uniform(s_sum[2 * PT_NW]), begin = pg_uniform(s_sum[2 * PT_NW + 1]), rows = pg_uniform(s_sum[2 * PT_NW + 2]);
  at.b = (int)own;
  if (at.b < 0) return false;  // (lengths changed under way: a program's error, but one that ends)
  at.lens = pt_lens{(int)rows, (int)(rows >> 32), (int)(own >> 32)};
  at.cost = pt_cost_of(A, at.lens);
  if (target) {
    const int k = (int)pg_uniform(pg_div(at.cost.each + target - 1, target)), nth = w - (int)begin, tile = nth / k, part = nth - tile * k;
    at.tile = tile;
    at.begin = 0;
    at.x0 = pg_uniform(pg_div(at.cost.each * part, k));
    at.x1 = pg_uniform(pg_div(at.cost.each * (part + 1), k));
    if (threadIdx.x == 0) {
      s_shares.w0 = w - part;
      s_shares.parts = k;
    }
  } else {
    at.tile = pg_uniform(pg_div(at.x0 - begin, at.cost.each));
    at.begin = begin + at.tile * at.cost.each;
  }
  return true;
}
// The next tile on the line; there is one, unless lengths changed under way (an error of the program's, but one that ends)
__device__ __forceinline__ bool pt_next(const pt_args& A, pt_place& at) {
  at.begin += at.cost.each;
  if (++at.tile < at.cost.tiles) return true;
  at.tile = 0;
  do {
    if (++at.b >= A.a.requests.n_requests) return false;
    at.lens = pt_lens_of(A.a.requests, at.b);
    at.cost = pt_cost_of(A, at.lens);
  } while (at.cost.tiles == 0);
  return true;
}
// The key at which a tile's part ends that ends at y of its cost: the same for the one that begins there.
__device__ __forceinline__ int pt_key_at(int64_t y, int64_t cost, int n) {
  if (y >= cost) return n;
  const int u = (int)((double)n * ((double)y / (double)cost));
  return __builtin_amdgcn_readfirstlane(u / PT_STEP * PT_STEP);
}

// What the join has to know of a part: whose it is, and which workgroups have the tile's others. Every workgroup leaves two of them, of the
// tile that began before its piece and of the one that ends behind it; parts 0: there is none.
struct __attribute__((aligned(16))) pt_record {
  int w0, parts;
  int t0, rows, hk0, block;
  int b, begin, end, kv;
  int pad[2];
};
__device__ __forceinline__ pt_record* pt_records(const pt_args& A, int wgs, int dp, int w) {
  return (pt_record*)((float*)A.a.work + (int64_t)wgs * 2 * A.heads * PT_ROWS * (dp + 4)) + 2 * w;
}

// Whether one of the bytes is set. All threads call.
__device__ __forceinline__ bool pt_any(const uint8_t* bytes, int n) {
  uint32_t any = 0;
  for (int i = threadIdx.x; i < n / 4; i += PT_NT) any |= ((const uint32_t*)bytes)[i];
  for (int i = n / 4 * 4 + threadIdx.x; i < n; i += PT_NT) any |= bytes[i];
  return __syncthreads_or(any != 0);
}

// One row key by key, by one wave: what a row holds that came out not finite. The average so far is held, not the sum: of finite values it
// is finite, however large they are.
template <int KT, int QT>
__device__ __forceinline__ void pt_row_again(const pt_args& A, const pg_request& r, int t, int h) {
  const sah_page_attention_args& P = A.a;
  const sah_page_cache& C = P.cache;
  constexpr int E = PG_MAX_D / SAH_WAVE;
  const int lane = threadIdx.x & (SAH_WAVE - 1), hk = h / (P.Hq / C.Hkv), shift = 31 - __builtin_clz(C.page_size);
  const int64_t p = r.base + t;
  const int hi = p < r.kv ? (int)p : r.kv - 1;
  const int32_t* list = P.pages ? P.pages + ((int64_t)t * C.Hkv + hk) * P.n_select : nullptr;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + e * SAH_WAVE;
    q[e] = d < C.D ? sah_load<QT>(P.q, (int64_t)t * P.qs_t + (int64_t)h * P.qs_h + d) : 0.f;
    acc[e] = 0.f;
  }
  const int entries = p < 0 || r.kv == 0 ? 0 : list ? P.n_select : (hi >> shift) + 1;
  for (int i = 0; i < entries; ++i) {
    const int lg = list ? list[i] : i;
    if (lg < 0 || lg >= P.requests.table_width || lg > hi >> shift) continue;
    const int page = P.requests.block_table[(int64_t)r.b * P.requests.table_pitch + lg];
    if (page < 0 || page >= C.n_pages) continue;
    for (int in = 0; in < C.page_size; ++in) {
      const int j = (lg << shift) + in;
      if (j > hi) break;
      if (P.window > 0 && j >= P.sink && j <= p - P.window) continue;
      const int64_t ka = page * C.ks_p + in * C.ks_t + hk * C.ks_h, va = page * C.vs_p + in * C.vs_t + hk * C.vs_h;
      float ks = 1.f, vs = 1.f;
      if (KT == SAH_E4M3) {
        const int64_t at = ((int64_t)page * C.Hkv + hk) * C.page_size + in;
        ks = pg_scale(C.k_scales[at]);
        vs = pg_scale(C.v_scales[at]);
      }
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane + e * SAH_WAVE;
        if (d < C.D) s = fmaf(q[e], pg_element<KT>(C.k, ka + d, ks), s);
      }
      s = sah_wave_sum(s) * P.scaling;
      const float m_new = fmaxf(m, s);
      if (m_new == -INFINITY && s == s) continue;  // (a NaN is no maximum, but the row's result)
      const float before = l * expf(m - m_new), w = expf(s - m_new);
      m = m_new;
      l = before + w;
      const float old = before / l, share = w / l;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane + e * SAH_WAVE;
        if (d < C.D) acc[e] = acc[e] * old + share * pg_element<KT>(C.v, va + d, vs);
      }
    }
  }
  const float seen = P.sinks && m != -INFINITY ? l / (l + expf(P.sinks[h] - m)) : 1.f;  // all but the sink's share
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + e * SAH_WAVE;
    if (d < C.D) sah_store<QT>(P.out, (int64_t)t * P.os_t + (int64_t)h * P.os_h + d, acc[e] * seen);
  }
}
// Whether a result is the type's finite number; rows with others are done again
template <int QT>
__device__ __forceinline__ bool pt_fine(float v) { return fabsf(v) < (QT == SAH_F32 ? INFINITY : QT == SAH_BF16 ? 0x1.ffp127f : 65520.f); }

// two 16-bit halves: the lower ones of a and b, or the upper ones
__device__ __forceinline__ uint32_t pt_low(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t pt_high(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// the largest, or the sum, of what lanes n, n + 16, n + 32 and n + 48 hold
__device__ __forceinline__ float pt_quad_max(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_permlane16_swap(sah_float_to_bits(v), sah_float_to_bits(v), false, false);
  v = fmaxf(sah_bits_to_float(r[0]), sah_bits_to_float(r[1]));
#endif
  return sah_half_max(v);
}
__device__ __forceinline__ float pt_quad_sum(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_permlane16_swap(sah_float_to_bits(v), sah_float_to_bits(v), false, false);
  v = sah_bits_to_float(r[0]) + sah_bits_to_float(r[1]);
#endif
  return sah_half_sum(v);
}

// x rounded to a term of MT's bits, two of them packed, and what is left of them
template <int MT>
__device__ __forceinline__ uint32_t pt_term(float& a, float& b) {
  uint32_t w = sah_pack2_hw<MT>(a, b);
  sah_keep(w);  // taken apart as it is, instead of converted a second time
  if (MT == SAH_BF16) {
    a -= sah_bits_to_float(w << 16);
    b -= sah_bits_to_float(w & 0xffff0000u);
  } else {
    a -= sah_f16_to_float((uint16_t)w);
    b -= sah_f16_to_float((uint16_t)(w >> 16));
  }
  return w;
}

__device__ __forceinline__ sah_f32x4 pt_mfma_f32(float a, float b, sah_f32x4 c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
#else
  return c;
#endif
}

// Workgroups of a CU, by the registers that an instance needs: waves of a SIMD
__host__ __device__ constexpr int pt_per_cu(int cache_type, int dim) {
  return cache_type == SAH_F32 ? (dim > 64 ? 1 : 2) : dim > 128 ? 1 : dim > 64 ? 2 : 3;
}

// From a uniform address and an offset of the lane: told apart here, or the compiler adds them up in vector registers.
template <typename W, bool ONCE = false>
__device__ __forceinline__ W pt_load(const void* base, uint32_t offset) {
  sah_keep(offset);
  const W* p = (const W*)((const char*)base + offset);
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  return *p;
}

// Where a 16-key tile (in small pages: a key) lies: bytes from a key head's first key and value, and scale; its number.
struct __attribute__((aligned(16))) pt_where {
  int64_t k, v, scale;
  int first, pad;
};

// SMALL: pages of less than 16 tokens, where a 16-key tile's keys do not lie in one page. ONCE: keys and values are read past the caches.
template <int KT, int QT, int DP, bool SMALL, bool ONCE>
__global__ __launch_bounds__(PT_NT, (pt_per_cu(KT, DP))) void k_page_attn(pt_args) {
  sah_touch_kernargs<sizeof(pt_args)>();
  typedef pt_types<KT, QT> T;
  constexpr int ES = pg_size(KT), MT = T::MT;
  constexpr int KL = DP * ES / 64;                                    // 16-byte loads of a lane and key tile
  constexpr int NC = KT == SAH_E4M3 ? DP / 16 : KT == SAH_F32 ? 4 : DP >= 128 ? 8 : 4;  // elements of a lane's piece of a value row
  constexpr int H = DP / (16 * NC);                                   // pieces
  constexpr int VW = NC * ES / 4;                                     // 32-bit words of a piece
  constexpr int TILES = DP / 16;
  constexpr int PITCH = DP + 4;                                       // floats of a row in LDS
  // key tiles of a wave's step: fp32 rows of 256 dims leave no registers for two
  constexpr int NA = KT == SAH_F32 && DP > 128 ? 1 : 2, STEP = 16 * NA;
  constexpr int MOST = SMALL ? PT_MOST / 4 : PT_MOST, SLOTS = SMALL ? MOST : MOST / 16;
  __shared__ pt_where s_at[SLOTS];                                    // of the 16-key tiles (SMALL: keys) that are worked on
  __shared__ __align__(16) float s_acc[PT_NW][PT_ROWS][PITCH];
  __shared__ float s_ml[PT_NW][2][PT_ROWS];
  __shared__ unsigned long long s_bad;  // a bit a head and row
  __shared__ int64_t s_sum[2 * PT_NW + 3];
  __shared__ pt_shares s_shares;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id(), i16 = lane & 15, g = lane >> 4;
  const int w = pt_number();
  pt_place at;
  const uint8_t* lost = pt_arguments().lost;
  if ((lost && !pt_any(lost, pt_arguments().n_lost)) || !pt_start(pt_arguments(), w, gridDim.x, s_sum, s_shares, at)) {
    if (threadIdx.x < 2) pt_records(pt_arguments(), gridDim.x, DP, w)[threadIdx.x].parts = 0;
    return;
  }
  int left = 0;  // records that have been written, a bit each
  int64_t x = at.x0;
  for (;;) {
    const pt_args& A = pt_arguments();
    const sah_page_attention_args& P = A.a;
    const sah_page_cache& C = P.cache;
    const int G = P.Hq / C.Hkv, shift = 31 - __builtin_clz(C.page_size);
    const float c_exp = pt_log2(P.scaling), sign = P.scaling < 0.f ? -1.f : 1.f;
    const int64_t y0 = x - at.begin, y1 = at.x1 - at.begin < at.cost.each ? at.x1 - at.begin : at.cost.each;
    const bool whole = y0 == 0 && y1 == at.cost.each;
    const int tile = __builtin_amdgcn_readfirstlane((int)at.tile);  // (n_tokens * Hq fits)
    const int head_groups = C.Hkv / A.heads, tb = tile / head_groups, hk0 = (tile - tb * head_groups) * A.heads, block = tb % A.blocks, i0 = tb / A.blocks * A.tokens;
    const int hk = hk0 + (wave & (A.heads - 1)), turns = PT_NW / A.heads, turn = wave / A.heads;  // this wave's head; a head's waves take turns
    const int t0 = at.lens.begin + i0;
    const pg_request req = pg_make(P.requests, C.page_size, at.b, at.lens.begin, at.lens.end, at.lens.kv);
    const int n_tok = A.tokens < req.n_new - i0 ? A.tokens : req.n_new - i0;
    const int rows = A.blocks > 1 ? (G - block * PT_ROWS < PT_ROWS ? G - block * PT_ROWS : PT_ROWS) : n_tok * G;
    const int64_t p_lo = req.base + t0, p_hi = p_lo + n_tok - 1;
    const pt_keys keys = pt_keys_of(A, req, p_lo, p_hi);
    const int u_first = y0 ? pt_key_at(y0, at.cost.each, keys.n) : 0, u_end = pt_key_at(y1, at.cost.each, keys.n);
    const bool live = i16 < rows;
    const int rr = live ? i16 : rows - 1;
    const int tok = t0 + (A.blocks > 1 ? 0 : rr / G), head = hk * G + (A.blocks > 1 ? block * PT_ROWS + rr : rr % G);
    const int64_t p = req.base + tok;
    const int last = p < keys.hi ? (p < -1 ? -1 : (int)p) : keys.hi;          // the last key that this lane's row sees
    const int least = p_lo < keys.hi ? (p_lo < -1 ? -1 : (int)p_lo) : keys.hi; // ... that all rows see
    // window: where it begins for this lane's row, for some row, for all rows
    const int sink = P.window ? P.sink : 0;
    auto window_from = [&](int64_t at_p) { return P.window && at_p >= P.window ? (int)(at_p - P.window + 1 < keys.hi + 1 ? at_p - P.window + 1 : keys.hi + 1) : 0; };
    const int from_own = window_from(p), from_any = window_from(p_lo), from_all = window_from(p_hi);
    if (threadIdx.x == 0) s_bad = 0;

    // Queries as the second operand, in the order in which a lane's 16 bytes of a key come: requested here, made into it when the first keys are
    // under way.
    constexpr int QS = KT == SAH_F32 ? KL : DP / 32, QE = KT == SAH_F32 ? 4 : 8, QW = QE * pg_size(QT) / 16;  // pieces, elements, loads of a piece
    const char* qp = (const char*)P.q + ((int64_t)tok * P.qs_t + (int64_t)head * P.qs_h) * pg_size(QT);
    uint4 qf[T::NQ][QS];
    sah_u4 q_raw[QS][QW];
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int d = KT == SAH_F32 ? 16 * s + 4 * g : KT == SAH_E4M3 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
#pragma unroll
      for (int i = 0; i < QW; ++i) {
        q_raw[s][i] = sah_u4{0, 0, 0, 0};
        if (d < C.D && live) q_raw[s][i] = *(const sah_u4*)(qp + d * pg_size(QT) + 16 * i);
      }
    }
    // Where the keys from u0 on lie, MOST of them
    auto look_up = [&](int u0) __attribute__((always_inline)) {
      const int u1 = u_end - u0 < MOST ? u_end : u0 + MOST;
      constexpr int EACH = SMALL ? 1 : 16;
      const int n_slots = (u1 - u0 + STEP - 1) / STEP * (STEP / EACH);
      const int32_t* list = P.pages ? P.pages + ((int64_t)t0 * C.Hkv + hk0) * P.n_select : nullptr;
      for (int s = threadIdx.x; s < n_slots; s += PT_NT) {
        const int u = u0 + s * EACH, e = u >> shift;
        int64_t in = u & (C.page_size - 1);
        int lg = e;
        if (list) lg = e < P.n_select ? list[e] : -1;
        else if (keys.skip && u >= keys.sinks) lg = e + (keys.skip >> shift);
        int64_t page = -1;
        if (lg >= 0 && lg < P.requests.table_width && lg <= keys.hi >> shift) page = P.requests.block_table[(int64_t)req.b * P.requests.table_pitch + lg];
        pt_where at;
        // a page that is not there: another one's keys, behind every position (table_width pages end before that)
        at.first = (int)(0x80000000u - (uint32_t)C.page_size + (uint32_t)in);
        if (page >= 0 && page < C.n_pages) at.first = (lg << shift) + (int)in;
        else page = in = 0;
        at.k = (page * C.ks_p + in * C.ks_t) * ES;
        at.v = (page * C.vs_p + in * C.vs_t) * ES;
        at.scale = page * C.Hkv * C.page_size + in;
        s_at[s] = at;
      }
    };
    __syncthreads();  // the sums of the tile before have been read
    if (u_first < u_end) look_up(u_first);
    {
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        float v[8];
#pragma unroll
        for (int i = 0; i < QW; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t x = q_raw[s][i][k];
            if constexpr (QT == SAH_F32) {
              v[4 * i + k] = sign * sah_bits_to_float(x);
            } else if constexpr (QT == SAH_BF16) {
              v[2 * k] = sign * sah_bits_to_float(x << 16);
              v[2 * k + 1] = sign * sah_bits_to_float(x & 0xffff0000u);
            } else {
              v[2 * k] = sign * sah_f16_to_float((uint16_t)x);
              v[2 * k + 1] = sign * sah_f16_to_float((uint16_t)(x >> 16));
            }
          }
        if constexpr (KT == SAH_F32) {
          qf[0][s] = make_uint4(sah_float_to_bits(v[0]), sah_float_to_bits(v[1]), sah_float_to_bits(v[2]), sah_float_to_bits(v[3]));
        } else {
#pragma unroll
          for (int i = 0; i < T::NQ; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pt_term<MT>(v[2 * k], v[2 * k + 1]);
            qf[i][s] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
    __syncthreads();

    float m_run = -INFINITY, l_run = 0.f;
    sah_f32x4 acc[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;

    // What lies behind a shorter head's end is its last piece again: the queries are 0 there, the results nobody's. Offsets of a lane from a
    // key tile's first key (SMALL: from its own key).
    uint32_t k_in[KL], v_in[H][4];
#pragma unroll
    for (int s = 0; s < KL; ++s) {
      const int in = 64 * s + 16 * g;
      k_in[s] = (uint32_t)((SMALL ? 0 : i16 * C.ks_t * ES) + (in < C.D * ES ? in : C.D * ES - 16));
    }
#pragma unroll
    for (int s = 0; s < H; ++s) {
      const int in = (s * 16 + i16) * NC;
#pragma unroll
      for (int v = 0; v < 4; ++v) v_in[s][v] = (uint32_t)((SMALL ? 0 : (4 * g + v) * C.vs_t * ES) + (in < C.D ? in : C.D - NC) * ES);
    }
    const char* kbase = (const char*)C.k + (int64_t)hk * C.ks_h * ES;
    const char* vbase = (const char*)C.v + (int64_t)hk * C.vs_h * ES;
    const uint8_t *k_scales = C.k_scales + (int64_t)hk * C.page_size, *v_scales = C.v_scales + (int64_t)hk * C.page_size;

    struct keys_of { sah_u4 r[NA][KL]; uint32_t scale[NA]; } kb;           // scales: bytes, of four keys, this lane's among them
    struct values_of { uint32_t r[H][4 * NA][VW]; uint32_t scale[NA]; } vb; // ... of the four whose values a lane has
    int u0 = u_first;                  // of what s_at holds
    auto fetch_k = [&](int u, keys_of& k) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        if constexpr (SMALL) {
          const pt_where& at = s_at[u + 16 * a + i16 - u0];
          const char* from = kbase + at.k;
          if constexpr (KT == SAH_E4M3) k.scale[a] = k_scales[at.scale] * 0x01010101u;
#pragma unroll
          for (int s = 0; s < KL; ++s) k.r[a][s] = *(const sah_u4*)(from + k_in[s]);
        } else {
          const pt_where& at = s_at[(u - u0) / 16 + a];
          const char* from = kbase + pg_uniform(at.k);
          if constexpr (KT == SAH_E4M3) k.scale[a] = pt_load<uint32_t>(k_scales + pg_uniform(at.scale), i16 & 12);
#pragma unroll
          for (int s = 0; s < KL; ++s) k.r[a][s] = pt_load<sah_u4, ONCE>(from, k_in[s]);
        }
      }
    };
    auto fetch_v = [&](int u, values_of& x) __attribute__((always_inline)) {
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        const char* from = nullptr;
        if constexpr (!SMALL) {
          const pt_where& at = s_at[(u - u0) / 16 + a];
          from = vbase + pg_uniform(at.v);
          if constexpr (KT == SAH_E4M3) x.scale[a] = pt_load<uint32_t>(v_scales + pg_uniform(at.scale), 4 * g);
        } else if constexpr (KT == SAH_E4M3) {
          x.scale[a] = 0;
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          if constexpr (SMALL) {
            const pt_where& at = s_at[u + 16 * a + 4 * g + v - u0];
            from = vbase + at.v;
            if constexpr (KT == SAH_E4M3) x.scale[a] |= (uint32_t)v_scales[at.scale] << (8 * v);
          }
#pragma unroll
          for (int s = 0; s < H; ++s) {
            uint32_t* to = x.r[s][4 * a + v];
            typedef uint32_t words __attribute__((ext_vector_type(VW)));
            const words w = SMALL ? *(const words*)(from + v_in[s][v]) : pt_load<words, ONCE>(from, v_in[s][v]);
#pragma unroll
            for (int i = 0; i < VW; ++i) to[i] = w[i];
          }
        }
      }
    };

    auto step = [&](int u, int next, keys_of& kx, values_of& vx) __attribute__((always_inline)) {
      sah_f32x4 s[NA];
#pragma unroll
      for (int a = 0; a < NA; ++a) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][e] = 0.f;
        const float scale = KT == SAH_E4M3 ? pg_scale_of(kx.scale[a], i16 & 3) : 1.f;
#pragma unroll
        for (int c = 0; c < KL; ++c) {
          const sah_u4 k = kx.r[a][c];
          if constexpr (KT == SAH_F32) {
            s[a] = pt_mfma_f32(sah_bits_to_float(k.x), sah_bits_to_float(qf[0][c].x), s[a]);
            s[a] = pt_mfma_f32(sah_bits_to_float(k.y), sah_bits_to_float(qf[0][c].y), s[a]);
            s[a] = pt_mfma_f32(sah_bits_to_float(k.z), sah_bits_to_float(qf[0][c].z), s[a]);
            s[a] = pt_mfma_f32(sah_bits_to_float(k.w), sah_bits_to_float(qf[0][c].w), s[a]);
          } else if constexpr (KT == SAH_E4M3) {
            const uint4 k0 = make_uint4(pg_widen2<false>(k.x, scale), pg_widen2<true>(k.x, scale), pg_widen2<false>(k.y, scale), pg_widen2<true>(k.y, scale));
            const uint4 k1 = make_uint4(pg_widen2<false>(k.z, scale), pg_widen2<true>(k.z, scale), pg_widen2<false>(k.w, scale), pg_widen2<true>(k.w, scale));
#pragma unroll
            for (int i = 0; i < T::NQ; ++i) {
              s[a] = sah_mfma_16x16x32<MT>(k0, qf[i][2 * c], s[a]);
              s[a] = sah_mfma_16x16x32<MT>(k1, qf[i][2 * c + 1], s[a]);
            }
          } else {
            s[a] = sah_mfma_16x16x32<MT>(make_uint4(k.x, k.y, k.z, k.w), qf[0][c], s[a]);
          }
        }
      }
      fetch_k(next, kx);
      // keys that not every row sees; values of keys that no row sees are made 0
      int first[NA] = {};
      bool plain = !SMALL;   // uniform
      if constexpr (!SMALL) {
#pragma unroll
        for (int a = 0; a < NA; ++a) {
          first[a] = __builtin_amdgcn_readfirstlane(s_at[(u - u0) / 16 + a].first);
          plain = plain & (first[a] + 15 <= least) & ((first[a] >= from_all) | (first[a] + 15 < sink));
        }
      }
      if (!plain) {
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = SMALL ? s_at[u + 16 * a + 4 * g + e - u0].first : first[a] + 4 * g + e;
            const bool on = (j <= last) & ((j >= from_own) | (j < sink)), some = (j <= keys.hi) & ((j >= from_any) | (j < sink));
            s[a][e] = on ? s[a][e] : -INFINITY;
#pragma unroll
            for (int c = 0; c < H; ++c)
#pragma unroll
              for (int w = 0; w < VW; ++w) vx.r[c][4 * a + e][w] = some ? vx.r[c][4 * a + e][w] : 0u;
            if constexpr (KT == SAH_E4M3) vx.scale[a] = some ? vx.scale[a] : vx.scale[a] & ~(0xffu << (8 * e));  // (0 times the byte 255 is NaN)
          }
      }
      float mx = s[0][0];
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[a][e]);
      mx = pt_quad_max(mx);
      // (-inf - -inf is NaN: no rise)
      if (__ballot((mx - m_run) * c_exp > T::SLACK) != 0) {
        const float m_new = fmaxf(m_run, mx);
        const float up = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * c_exp);
        m_run = m_new;
        l_run *= up;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][e] *= up;
      }
      // (Products are compared and subtracted before they are scaled: a product times c_exp, rounded, beside the same unrounded leaves a difference of
      // its own size where products are large.)
      const float m_at = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[a][e] = __builtin_amdgcn_exp2f(fmaf(s[a][e] - m_at, c_exp, T::SCALE));
          l_run += s[a][e];
        }
      if constexpr (KT == SAH_F32) {
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < H; ++c)
#pragma unroll
              for (int w = 0; w < NC; ++w) acc[c * NC + w] = pt_mfma_f32(sah_bits_to_float(vx.r[c][4 * a + e][w]), s[a][e], acc[c * NC + w]);
      } else {
        uint32_t term[T::NP][4];
        float rest[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[e] = s[e / 4][e % 4];
#pragma unroll
        for (int i = 0; i < T::NP; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) term[i][k] = pt_term<MT>(rest[2 * k], rest[2 * k + 1]);
#pragma unroll
        for (int c = 0; c < H; ++c)
#pragma unroll
          for (int pair = 0; pair < NC / 2; ++pair) {
            uint32_t two[8];  // the pair's dims of the 8 keys
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              if constexpr (KT == SAH_E4M3) {
                const float scale = pg_scale_of(vx.scale[k / 4], k % 4);
                two[k] = pair % 2 ? pg_widen2<true>(vx.r[c][k][pair / 2], scale) : pg_widen2<false>(vx.r[c][k][pair / 2], scale);
              } else {
                two[k] = vx.r[c][k][pair];
              }
            }
            const uint4 lo = make_uint4(pt_low(two[0], two[1]), pt_low(two[2], two[3]), pt_low(two[4], two[5]), pt_low(two[6], two[7]));
            const uint4 hi = make_uint4(pt_high(two[0], two[1]), pt_high(two[2], two[3]), pt_high(two[4], two[5]), pt_high(two[6], two[7]));
#pragma unroll
            for (int i = 0; i < T::NP; ++i) {
              const uint4 w = make_uint4(term[i][0], term[i][1], term[i][2], term[i][3]);
              acc[c * NC + 2 * pair] = sah_mfma_16x16x32<MT>(lo, w, acc[c * NC + 2 * pair]);
              acc[c * NC + 2 * pair + 1] = sah_mfma_16x16x32<MT>(hi, w, acc[c * NC + 2 * pair + 1]);
            }
          }
      }
      fetch_v(next, vx);
    };
    for (; u0 < u_end; u0 += MOST) {  // (uniform; the next one's first key fits 32 bits: the host has checked what a request can have)
      const int u1 = u_end - u0 < MOST ? u_end : u0 + MOST;
      if (u0 != u_first) {
        __syncthreads();  // the places before have been read
        look_up(u0);
        __syncthreads();
      }
      const int round = STEP * turns;
      int u = u0 + STEP * turn;
      if (u >= u1) continue;
      // Behind a wave's last step it is requested again, from the caches: a way through the loop that skips a request would have the compiler wait
      // for all of them.
      const int end = u + (u1 - 1 - u) / round * round;
      fetch_k(u, kb);
      fetch_v(u, vb);
      for (; u < u1; u += round) step(u, u < end ? u + round : end, kb, vb);
    }

    // the four waves' sums, row by row in LDS
    l_run = pt_quad_sum(l_run);
    if (live) {
      if (g == 0) {
        s_ml[wave][0][i16] = m_run;
        s_ml[wave][1][i16] = l_run;
      }
#pragma unroll
      for (int c = 0; c < H; ++c)
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int e = 0; e < NC; e += 4)
            *(float4*)&s_acc[wave][i16][(c * 16 + 4 * g + v) * NC + e] =
                make_float4(acc[c * NC + e][v], acc[c * NC + e + 1][v], acc[c * NC + e + 2][v], acc[c * NC + e + 3][v]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < A.heads * rows * (DP / 4); i += PT_NT) {
      const int of = i / (DP / 4), d = 4 * (i % (DP / 4)), hh = of / rows, r = of - hh * rows;
      float m = -INFINITY, l = 0.f;
      for (int w = hh; w < PT_NW; w += A.heads) m = fmaxf(m, s_ml[w][0][r]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = hh; w < PT_NW; w += A.heads) {
        const float mw = s_ml[w][0][r], lw = s_ml[w][1][r], up = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - m) * c_exp);
        l += lw == lw ? lw * up : lw;  // (a wave whose sum is NaN has no maximum, perhaps)
        const float4 a = *(const float4*)&s_acc[w][r][d];
        o.x += a.x * up;
        o.y += a.y * up;
        o.z += a.z * up;
        o.w += a.w * up;
      }
      const int rt = t0 + (A.blocks > 1 ? 0 : r / G), rh = (hk0 + hh) * G + (A.blocks > 1 ? block * PT_ROWS + r : r % G);
      if (!whole) {  // a part: to slot 0 where the tile began before this workgroup's piece, else to slot 1
        float* to = (float*)P.work + ((((int64_t)w * 2 + (y0 ? 0 : 1)) * A.heads + hh) * PT_ROWS + r) * (DP + 4);
        if (d == 0) *(float2*)to = make_float2(m, l);
        *(float4*)(to + 4 + d) = o;
        continue;
      }
      bool fine = l == l;
      if (P.sinks && m != -INFINITY) l += __builtin_amdgcn_exp2f(fmaf(P.sinks[rh], 1.4426950408889634f, T::SCALE) - m * c_exp);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
      if (d >= C.D) continue;
      fine = fine && pt_fine<QT>(o.x) && pt_fine<QT>(o.y) && pt_fine<QT>(o.z) && pt_fine<QT>(o.w);
      if (!fine) atomicOr(&s_bad, 1ull << (hh * PT_ROWS + r));
      char* to = (char*)P.out + ((int64_t)rt * P.os_t + (int64_t)rh * P.os_h + d) * pg_size(QT);
      if (QT == SAH_F32) *(float4*)to = o;
      else *(uint2*)to = make_uint2(sah_pack2_hw<QT>(o.x, o.y), sah_pack2_hw<QT>(o.z, o.w));
    }
    if (!whole && wave == PT_NW - 1) {
      const pt_shares shares = s_shares;
      const int64_t key = at.begin + (lane < 32 ? 0 : at.cost.each - 1);
      int w0 = shares.w0, w1 = shares.w0 + shares.parts - 1;
      if (shares.parts == 0) shares.holders(key, key - at.x0, w, w0, w1);
      pt_record rec{};
      rec.w0 = w0 > 0 ? (w0 < w ? w0 : w) : 0;
      rec.parts = (w1 > w ? (w1 < (int)gridDim.x ? w1 : (int)gridDim.x - 1) : w) - rec.w0 + 1;
      rec.t0 = t0; rec.rows = rows; rec.hk0 = hk0; rec.block = block;
      rec.b = at.b; rec.begin = at.lens.begin; rec.end = at.lens.end; rec.kv = at.lens.kv;
      if (lane == 0) pt_records(A, gridDim.x, DP, w)[y0 ? 0 : 1] = rec;
    }
    left |= whole ? 0 : y0 ? 1 : 2;
    if (whole) {
      __syncthreads();
      unsigned long long bad = s_bad;  // rows that are not finite are done again, each by a wave
      for (int i = 0; bad; ++i) {
        const int hh = __builtin_ctzll(bad) / PT_ROWS, r = __builtin_ctzll(bad) % PT_ROWS;
        bad &= bad - 1;
        if (i % PT_NW != wave) continue;
        pt_row_again<KT, QT>(A, req, t0 + (A.blocks > 1 ? 0 : r / G), (hk0 + hh) * G + (A.blocks > 1 ? block * PT_ROWS + r : r % G));
      }
      if (at.begin + y1 < at.x1) __syncthreads();  // (s_bad has been read)
    }
    x = at.begin + y1;
    if (x >= at.x1 || !pt_next(pt_arguments(), at)) break;
  }
  if (threadIdx.x < 2 && !(left >> threadIdx.x & 1)) pt_records(pt_arguments(), gridDim.x, DP, w)[threadIdx.x].parts = 0;
}

// Joins the parts of tiles' rows: sum over parts of 2^((m_part - m) c) (l, acc), then acc / l. The workgroups that had a tile's parts deal its rows out
// among themselves; DP / 4 lanes hold a row's dims, and where a workgroup has fewer rows than such groups of lanes, a row's parts are shared by several. blockIdx.y: the
// tile that began before the workgroup's piece, or the one that ends behind it. Two
// trips to memory, the record's and the parts' (4 us; 128 parts a row, 32768 keys of one answer: 6.4). A join that finds a tile's place from the
// lengths takes 2 to 4 us more, one by the last workgroup of a tile would need counters that are zero before the call.
template <int KT, int QT, int DP>
__global__ __launch_bounds__(PT_NT) void k_page_attn_join(pt_args A) {
  sah_touch_kernargs<sizeof(pt_args)>();
  const sah_page_attention_args& P = A.a;
  const sah_page_cache& C = P.cache;
  typedef pt_types<KT, QT> T;
  constexpr int L = DP / 4, GROUPS = PT_NT / L, U = 8;
  __shared__ __align__(16) float4 s_acc[GROUPS][L];
  __shared__ float2 s_ml[GROUPS];
  const int l = threadIdx.x % L, group = threadIdx.x / L, w = pt_number();
  const pt_record rec = pt_records(A, gridDim.x, DP, w)[blockIdx.y];
  const int parts = rec.parts, w0 = rec.w0, all_rows = A.heads * rec.rows, nth_part = w - w0;
  if (parts == 0 || nth_part >= all_rows) return;
  const int rows = (all_rows - nth_part + parts - 1) / parts;  // this workgroup's: every parts-th
  int shared_by = 1;     // groups that share a row
  while (2 * shared_by * rows <= GROUPS) shared_by *= 2;
  const float* from = (const float*)P.work + (int64_t)w0 * 2 * A.heads * PT_ROWS * (DP + 4);
  const int G = P.Hq / C.Hkv;
  const float c_exp = pt_log2(P.scaling);
  float m, sum;
  float4 o;
  auto add = [&](float2 ml, const float4& v) __attribute__((always_inline)) {
    const float m_new = fmaxf(m, ml.x);
    const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * c_exp);
    const float z = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - m_new) * c_exp);
    // (a part whose sum is NaN has no maximum, perhaps: the row is done again all the same)
    sum = sum * a + (ml.y == ml.y ? ml.y * z : ml.y);
    m = m_new;
    o.x = o.x * a + v.x * z;
    o.y = o.y * a + v.y * z;
    o.z = o.z * a + v.z * z;
    o.w = o.w * a + v.w * z;
  };
  for (int r0 = 0; r0 < rows; r0 += GROUPS / shared_by) {  // uniform
    const int nth = r0 + group / shared_by, turn = group % shared_by, of_all = nth * parts + nth_part, hh = of_all / rec.rows, r = of_all - hh * rec.rows;
    const bool mine = nth < rows;
    m = -INFINITY;
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = turn; mine && p0 < parts; p0 += U * shared_by) {  // several parts requested at once; behind the last one it is taken again, and not added
      float2 ml[U];
      float4 v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int of = p0 + i * shared_by < parts ? p0 + i * shared_by : parts - 1;
        const float* part = from + (((int64_t)(of ? 2 * of : 1) * A.heads + hh) * PT_ROWS + r) * (DP + 4);
        ml[i] = *(const float2*)part;
        v[i] = *(const float4*)(part + 4 + 4 * l);
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (p0 + i * shared_by < parts) add(ml[i], v[i]);
    }
    if (shared_by > 1) {  // (then this is the only round)
      s_acc[group][l] = o;
      if (l == 0) s_ml[group] = make_float2(m, sum);
      __syncthreads();
      if (mine && turn == 0)
        for (int i = 1; i < shared_by; ++i) add(s_ml[group + i], s_acc[group + i][l]);
    }
    const bool ends = mine && turn == 0;
    const int hk = rec.hk0 + hh, rt = rec.t0 + (A.blocks > 1 ? 0 : r / G), rh = hk * G + (A.blocks > 1 ? rec.block * PT_ROWS + r : r % G), d = 4 * l;
    bool fine = true;
    if (ends) {
      fine = sum == sum;
      if (P.sinks && m != -INFINITY) sum += __builtin_amdgcn_exp2f(fmaf(P.sinks[rh], 1.4426950408889634f, T::SCALE) - m * c_exp);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (d < C.D) {
        o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
        fine = fine && pt_fine<QT>(o.x) && pt_fine<QT>(o.y) && pt_fine<QT>(o.z) && pt_fine<QT>(o.w);
        char* to = (char*)P.out + ((int64_t)rt * P.os_t + (int64_t)rh * P.os_h + d) * pg_size(QT);
        if (QT == SAH_F32) *(float4*)to = o;
        else *(uint2*)to = make_uint2(sah_pack2_hw<QT>(o.x, o.y), sah_pack2_hw<QT>(o.z, o.w));
      }
    }
    // rows that are not finite are done again, one after the other, by the wave that has them
    uint64_t again = __ballot(!fine);
    while (again) {
      const int at = __builtin_ctzll(again) / L * L;
      again &= L == SAH_WAVE ? 0ull : ~(((1ull << L) - 1) << at);
      pt_row_again<KT, QT>(A, pg_make(P.requests, C.page_size, rec.b, rec.begin, rec.end, rec.kv), __builtin_amdgcn_readlane(rt, at),
                           __builtin_amdgcn_readlane(rh, at));
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// What the contexts' keys and values may come to, by what the caller says
static double pt_context_bytes(const sah_page_attention_args& a) {
  double keys = (double)a.requests.table_width * a.cache.page_size;
  if (a.max_context > 0 && a.max_context < keys) keys = a.max_context;
  if (a.window && (double)a.sink + a.window < keys) keys = (double)a.sink + a.window;
  return keys * a.requests.n_requests * a.cache.Hkv * a.cache.D * 2 * pg_size(a.cache.dtype);
}

static pt_args pt_plan(const sah_page_attention_args* a, int& wgs) {
  pt_args A;
  A.a = *a;
  A.n_lost = 0;
  A.lost = nullptr;
  const int G = a->Hq / a->cache.Hkv;
  A.tokens = a->pages || G >= PT_ROWS ? 1 : PT_ROWS / G;
  A.blocks = (G + PT_ROWS - 1) / PT_ROWS;
  A.unit = a->cache.page_size > PT_STEP ? a->cache.page_size : PT_STEP;
  A.least = PT_LEAST / pg_size(a->cache.dtype);
  A.heads = a->pages || a->cache.Hkv % 2 ? 1 : a->cache.Hkv % 4 || pt_context_bytes(*a) <= PT_LAST_CACHE ? 2 : 4;
  // About as many workgroups as the call has work for, at most what the card holds at once. Only how the work is shared depends on it.
  const int64_t table = (int64_t)a->requests.table_width * a->cache.page_size;
  int64_t keys = table;
  if (a->pages) {
    keys = (int64_t)a->n_select * a->cache.page_size;
  } else {
    if (a->max_context > 0 && a->max_context < keys) keys = a->max_context;
    if (a->window && (int64_t)a->sink + a->window + 2 * (int64_t)A.unit < keys) keys = (int64_t)a->sink + a->window + 2 * (int64_t)A.unit;
  }
  const double tiles = ((double)a->requests.n_tokens / A.tokens + (A.tokens > 1 ? a->requests.n_requests : 0)) * A.blocks * a->cache.Hkv;
  const double n = tiles * (double)(keys + PT_TILE_COST) / A.least;
  const int most = PT_CUS * pt_per_cu(a->cache.dtype, a->cache.D);
  wgs = n < most ? ((int)n / PT_XCDS + 1) * PT_XCDS : most;
  return A;
}

// Chunks of an 8-bit cache: bytes of the copies of K and V and of their table, and the call on them; 0 where the cache is attended to as it is. A copy
// for wide tiles costs some 1.2 ns a key (8 heads of 128), and saves 8 ps for each row and key that it sees: worth it from 128 rows or so a request and key
// head on, with a window from so many times the context as it hides (32 heads on 8, us as it is / by a copy: 4 requests of 8192 keys, 64 rows 56 / 72,
// 128 rows 74 / 84, 256 rows 124 / 99, 512 rows 222 / 137; of those keys 512 + 128 seen, 1024 rows 56 / 70, 4096 rows 191 / 129; 2 requests of
// 32768, 2048 + 128 seen, 1024 rows 84 / 129, 4096 rows 248 / 175). Never for fp32 q: its terms go at the 16-bit matrix rate here, an fp32 copy at a
// tenth of it (4 requests of 8192 keys, 128 rows 80 / 268, 2048 rows 947 / 2952).
// A copy has room for the table's tokens of every request while this comes to no more than 256 MiB, else for max_context ones, where that is given. Tables are as
// wide as a server's longest request may become (16 of 131072 tokens, 8 heads of 128: 8 GiB): from 2 GiB on contexts are copied one behind the other, into as many
// pages as the cache has, 2 GiB at most. (A smaller room saves no time: 4 requests of 64 tokens over 8192 keys in tables of 16384 98 us, with room for 8192 and asking
// whether that was enough 107. 2048 tokens of one request over 16384 keys, 32 tables of 18432: 662 us; as it is 1699, alone in its table 658.)
//
// fp16 does not hold all that an 8-bit cache can, a context may be longer than max_context says, and all of them may need more room than there is: the copy's
// workgroups tell where that is so, and the cache is then attended to as it is, all rows once more (copies that hold everything pay for it with two launches that end at
// once: 4 requests of 64 fp16 tokens over 8192 keys 104 -> 113 us).
#define PT_COPY_BYTES 0x1p31
#define PT_COPY_WHOLE 0x1p28
struct pt_copy {
  int64_t bytes;    // K, V, their table, places and what was lost; 0: none
  int width;        // pages of a request, at most
  int64_t pages;    // of all
  int64_t table_at, placed_at, lost_at;  // placed_at: first pages and lengths, where contexts lie one behind the other, else 0
  int n_lost;       // 0: the copy holds everything
};
static pt_copy pt_copy_of(const sah_page_attention_args* a) {
  pt_copy c = {};
  if (a->pages || a->cache.dtype != SAH_E4M3 || a->dtype == SAH_F32) return c;
  const int table = a->requests.table_width, page_size = a->cache.page_size, n = a->requests.n_requests;
  const double keys = (double)table * page_size, reach = (double)a->sink + a->window, seen = a->window && reach < keys ? reach : keys;
  const double rows = (double)a->requests.n_tokens * (a->Hq / a->cache.Hkv);
  if (rows * seen <= 128 * keys * n) return c;
  const int64_t hint = ((int64_t)a->max_context + page_size - 1) / page_size;
  const double page = (double)page_size * a->cache.Hkv * a->cache.D * pg_size(a->dtype) * 2;
  c.width = hint > 0 && hint < table && (double)n * table * page > PT_COPY_WHOLE ? (int)hint : table;
  c.pages = (int64_t)n * c.width;
  if (c.pages * 4.0 > PT_COPY_BYTES / 8) return c;  // (their table)
  const bool placed = c.pages * page > PT_COPY_BYTES;
  if (placed) {
    const int64_t room = (int64_t)(PT_COPY_BYTES / page), least = a->cache.n_pages < room ? a->cache.n_pages : room;
    if (least < c.pages) c.pages = least;
    if (c.pages == 0) return c;
  }
  auto round = [](int64_t v) { return (v + 15) / 16 * 16; };
  c.table_at = c.pages * (int64_t)page;
  c.placed_at = placed ? round(c.table_at + (int64_t)n * c.width * 4) : 0;
  c.lost_at = placed ? round(c.placed_at + (int64_t)n * 8) : round(c.table_at + (int64_t)n * c.width * 4);
  const int64_t wgs = pg_load_workgroups(a->cache, a->requests, c.width * page_size);
  if (!wgs) return c;
  c.n_lost = a->dtype == SAH_F16 || c.width < table || placed ? (int)wgs : 0;
  c.bytes = round(c.lost_at + c.n_lost);
  return c;
}
static sah_paged_attention_args pt_on_copy(const sah_page_attention_args* a, const pt_copy& copy) {
  const sah_page_cache& c = a->cache;
  sah_paged_attention_args p = {};
  const int64_t row = c.D, token = row * c.Hkv, page = token * c.page_size;
  char* k = (char*)a->work;
  p.q = a->q; p.qs_t = a->qs_t; p.qs_h = a->qs_h;
  p.k = k; p.ks_p = page; p.ks_t = token; p.ks_h = row;
  p.v = k + copy.table_at / 2; p.vs_p = page; p.vs_t = token; p.vs_h = row;
  p.block_table = (const int32_t*)(k + copy.table_at);
  p.table_pitch = p.table_width = copy.width;
  p.kv_lens = copy.placed_at ? (const int32_t*)(k + copy.placed_at) + a->requests.n_requests : a->requests.kv_lens;
  p.cu_new = a->requests.cu_new;
  p.sinks = a->sinks;
  p.dtype = a->dtype;
  p.n_requests = a->requests.n_requests; p.n_tokens = a->requests.n_tokens; p.Hq = a->Hq; p.Hkv = c.Hkv; p.D = c.D;
  p.n_pages = (int)copy.pages; p.page_size = c.page_size;
  p.max_context = a->max_context; p.sink = a->sink; p.window = a->window;
  p.scaling = a->scaling;
  p.out = a->out; p.os_t = a->os_t; p.os_h = a->os_h;
  p.stream = a->stream;
  return p;
}

static int pt_dim(const sah_page_attention_args* a) { return a->cache.D <= 64 ? 64 : a->cache.D <= 128 ? 128 : 256; }

extern "C" int64_t sah_page_attention_work_bytes(const sah_page_attention_args* a) {
  if (!a || a->requests.n_tokens <= 0 || a->requests.n_requests <= 0 || a->requests.table_width <= 0 || a->cache.Hkv <= 0 || a->Hq < a->cache.Hkv ||
      a->cache.D <= 0 || a->cache.D > PG_MAX_D || a->cache.page_size <= 0 || (a->pages && a->n_select <= 0))
    return 0;
  int wgs;
  const pt_args A = pt_plan(a, wgs);
  const int64_t own = (int64_t)wgs * 2 * (A.heads * PT_ROWS * (pt_dim(a) + 4) * 4 + (int64_t)sizeof(pt_record));
  const pt_copy copy = pt_copy_of(a);
  if (!copy.bytes) return own;
  const sah_paged_attention_args p = pt_on_copy(a, copy);
  const int64_t others = 4 * sah_paged_attention_work_floats(&p);
  return copy.bytes + (copy.n_lost && own > others ? own : others);  // (one after the other)
}

// Whether keys and values are read past the caches: where every key is one tile's alone and the contexts, as far as the caller says, are twice what the
// last cache holds. (64 answers over 2.2 GB: 404 -> 384 us. Where the caches hold something, as 134 MB of 8 answers or keys that several tokens list, they
// gain: 32 us against 34, 59 against 94.)
static bool pt_once(const pt_args& A) {
  const sah_page_attention_args& a = A.a;
  if (a.pages || A.blocks > 1 || a.requests.n_tokens > (int64_t)a.requests.n_requests * A.tokens) return false;
  return pt_context_bytes(a) > PT_LAST_CACHE * 2;
}

template <int KT, int QT, int DP>
static int pt_launch(const pt_args& A, int wgs) {
  hipStream_t st = (hipStream_t)A.a.stream;
  {
    sah_timed timed("k_page_attn", A.a.stream);
    if (A.a.cache.page_size < 16) hipLaunchKernelGGL((k_page_attn<KT, QT, DP, true, false>), dim3(wgs), dim3(PT_NT), 0, st, A);
    else if (KT == SAH_E4M3 && pt_once(A)) hipLaunchKernelGGL((k_page_attn<KT, QT, DP, false, KT == SAH_E4M3>), dim3(wgs), dim3(PT_NT), 0, st, A);
    else hipLaunchKernelGGL((k_page_attn<KT, QT, DP, false, false>), dim3(wgs), dim3(PT_NT), 0, st, A);
    if (int rc = sah_launch_status("sah_page_attention")) return rc;
  }
  sah_timed timed("k_page_attn_join", A.a.stream);
  hipLaunchKernelGGL((k_page_attn_join<KT, QT, DP>), dim3(wgs, 2), dim3(PT_NT), 0, st, A);
  return sah_launch_status("sah_page_attention(join)");
}
template <int KT, int QT>
static int pt_launch_dim(const pt_args& A, int wgs) {
  const int dp = pt_dim(&A.a);
  return dp == 64 ? pt_launch<KT, QT, 64>(A, wgs) : dp == 128 ? pt_launch<KT, QT, 128>(A, wgs) : pt_launch<KT, QT, 256>(A, wgs);
}

extern "C" int sah_page_attention(const sah_page_attention_args* given) {
  static const char* what = "sah_page_attention";
  if (!given) return sah_fail(SAH_ENULL, "sah_page_attention: args is NULL");
  sah_page_attention_args own = *given;
  sah_page_attention_args* a = &own;
  sah_page_cache& c = a->cache;
  const sah_page_requests& r = a->requests;
  if (a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16) return sah_fail(SAH_EDTYPE, "sah_page_attention: dtype %d", a->dtype);
  if (int rc = pg_check_cache(c, true, what)) return rc;
  if (c.dtype != SAH_E4M3 && c.dtype != a->dtype) return sah_fail(SAH_EDTYPE, "sah_page_attention: dtype %d over a cache of dtype %d", a->dtype, c.dtype);
  if (a->Hq <= 0 || a->Hq % c.Hkv || a->max_context < 0 || a->sink < 0 || a->window < 0 || a->n_select < 0)
    return sah_fail(SAH_EINVAL, "sah_page_attention: bad sizes (heads %d / %d, max_context %d, sink %d, window %d, n_select %d)", a->Hq, c.Hkv, a->max_context,
                    a->sink, a->window, a->n_select);
  // (lists of no tokens lie nowhere)
  if (a->pages ? a->n_select == 0 : a->n_select > 0 && r.n_tokens > 0) return sah_fail(SAH_EINVAL, "sah_page_attention: pages and n_select go together");
  if (a->n_select && (a->window || a->sink)) return sah_fail(SAH_EINVAL, "sah_page_attention: pages and a window do not go together");
  if (!a->n_select && c.dtype != SAH_E4M3) return sah_fail(SAH_EDTYPE, "sah_page_attention: neither pages nor an 8-bit cache: sah_paged_attention's");
  if (int rc = pg_check_requests(r, c.page_size, true, what)) return rc;
  if ((int64_t)a->n_select * c.page_size > INT32_MAX - 4096) return sah_fail(SAH_ESHAPE, "sah_page_attention: n_select * page_size passes 2^31 - 4097");
  if ((int64_t)r.n_tokens * a->Hq > 1 << 30) return sah_fail(SAH_ESHAPE, "sah_page_attention: n_tokens * Hq passes 2^30");
  // the line of work is divided in doubles, also where running sums overlap
  const double each = (a->pages ? (double)a->n_select : (double)r.table_width) * c.page_size + PT_TILE_COST;
  if (((double)r.n_tokens + r.n_requests) * a->Hq * each * r.n_requests > 0x1p52) return sah_fail(SAH_ESHAPE, "sah_page_attention: too much work for one call");
  if (r.n_tokens == 0) return SAH_OK;
  if (!a->q || !a->out) return sah_fail(SAH_ENULL, "sah_page_attention: NULL pointer");
  if (r.n_tokens == 1) a->qs_t = a->os_t = 0;
  if (a->Hq == 1) a->qs_h = a->os_h = 0;
  const int es = pg_size(a->dtype);
  if (((uint64_t)a->q | (uint64_t)a->out | (uint64_t)a->work | (uint64_t)(es * (a->qs_t | a->qs_h | a->os_t | a->os_h))) % 16)
    return sah_fail(SAH_EINVAL, "sah_page_attention: addresses and strides must be multiples of 16 bytes");
  if (!sah_rows_apart<2>(c.D, {a->os_t, a->os_h}, {r.n_tokens, a->Hq})) return sah_fail(SAH_EINVAL, "sah_page_attention: rows of out overlap");
  if (!(a->scaling - a->scaling == 0.f)) return sah_fail(SAH_EINVAL, "sah_page_attention: scaling is not finite");
  const int64_t need = sah_page_attention_work_bytes(a);
  if (need && (!a->work || a->work_bytes < need)) return sah_fail(SAH_ECAPACITY, "sah_page_attention: work is too small");
  // rows are read again after others have been written
  const sah_span out = sah_span_of<2>(a->out, es, c.D, {a->os_t, a->os_h}, {r.n_tokens, a->Hq});
  if (sah_out_on_queries(a->q, a->qs_t, a->qs_h, a->out, a->os_t, a->os_h, r.n_tokens, a->Hq, c.D, es))
    return sah_fail(SAH_EINVAL, "sah_page_attention: out shares memory with q");
  if (pg_on_cache(out, c) || pg_on_requests(out, r, true) ||
      (a->pages && sah_meet(out, pg_span(a->pages, r.n_tokens, c.Hkv, a->n_select, 4))) ||
      (a->sinks && sah_meet(out, sah_span_of<1>(a->sinks, 4, 1, {1}, {a->Hq}))))
    return sah_fail(SAH_EINVAL, "sah_page_attention: out lies within the cache, the table, the lists or the lengths");
  int wgs;
  pt_args A = pt_plan(a, wgs);
  const pt_copy copy = pt_copy_of(a);
  if (copy.bytes) {
    sah_paged_attention_args p = pt_on_copy(a, copy);
    const int64_t row = c.D, token = row * c.Hkv, request = token * c.page_size * copy.width;
    char* work = (char*)a->work;
    int32_t* first = copy.placed_at ? (int32_t*)(work + copy.placed_at) : nullptr;
    A.n_lost = copy.n_lost;
    if (copy.n_lost) A.lost = (const uint8_t*)work + copy.lost_at;
    if (first) {
      if (int rc = pg_place(r, c.page_size, copy.width, copy.pages, first, first + r.n_requests, a->stream, what)) return rc;
    }
    const pg_load_out to{(void*)p.k, (void*)p.v, request, row, token, copy.width * c.page_size, (int32_t*)p.block_table, (uint8_t*)A.lost, first};
    if (int rc = pg_load(c, r, a->dtype, to, a->stream, what)) return rc;
    p.work = (float*)((char*)a->work + copy.bytes);
    p.work_floats = (a->work_bytes - copy.bytes) / 4;
    if (int rc = sah_paged_attention(&p)) return rc;
    if (!copy.n_lost) return SAH_OK;
    A.a.work = p.work;
  }
  if (c.dtype == SAH_F32) return pt_launch_dim<SAH_F32, SAH_F32>(A, wgs);
  if (c.dtype == SAH_BF16) return pt_launch_dim<SAH_BF16, SAH_BF16>(A, wgs);
  if (c.dtype == SAH_F16) return pt_launch_dim<SAH_F16, SAH_F16>(A, wgs);
  if (a->dtype == SAH_F32) return pt_launch_dim<SAH_E4M3, SAH_F32>(A, wgs);
  if (a->dtype == SAH_BF16) return pt_launch_dim<SAH_E4M3, SAH_BF16>(A, wgs);
  return pt_launch_dim<SAH_E4M3, SAH_F16>(A, wgs);
}
