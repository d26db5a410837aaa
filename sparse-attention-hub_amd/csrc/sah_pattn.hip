// Attention of new tokens over a key-value cache in pages, on the matrix cores.
//
// Of a request's new tokens and a key head's query heads every (token, head) is a row; 32 or 128 rows are a tile, which reads its
// keys once. All tiles of all requests, one after the other, are one line of work (measured in keys); every workgroup takes
// an equal piece of it, whatever the requests' lengths, finds its place from the lengths on the device, and works through
// tiles and parts of tiles. A part's (m, l, acc) goes to the workspace, a second kernel joins the parts of a tile.
//
// A wave owns 32 rows: S^T = K Q^T puts row j in lanes j and j + 32 (16 of 32 keys each), so a row's maximum and sum need one exchange
// between two lanes, and its weights are where the second product, O^T = V^T P^T, wants its B operand, with the key slots of a
// 16-key step taken in the order [0-3][8-11] / [4-7][12-15]. fp32: the 32 x 32 x 2 form, whose operands are single elements.
// Masked logits are replaced, not added to, so what a hidden key holds cannot reach them; keys that are not there (behind
// the request's last, or on a missing page) are staged from one that is. A visible row's product with a value that is
// not finite reaches the rows of its tile that do not see it (0 times it): rows that come out not finite are done again, key by key.
#include "sah_common.h"
#include "sah_spans.h"
#include "../../include/sah_serve.h"

#define PA_MAX_D 256
#define PA_CUS 256
#define PA_XCDS 8
// 16-byte pieces of staged keys that are read while as many are multiplied (2048 tokens over 18432 keys: 636 us; 4: 647, 8: 650)
// and 32-dim tiles of values (1, 2 and 4 alike)
#define PA_LOOK 2
#define PA_LOOK_V 2

// Shape of a launch. RW waves share the keys of a stage, each with 32 rows; RW = 1: every wave has keys of its own.
template <int DT, int DP, bool WIDE>
struct pa_shape {
  static constexpr int ES = DT == SAH_F32 ? 4 : 2;
  static constexpr int ROW = DP * ES;                      // bytes of a staged key
  static constexpr int NW = WIDE ? 4 : ROW <= 256 ? 8 : 2048 / ROW;
  static constexpr int NT = NW * SAH_WAVE;
  static constexpr int RW = WIDE ? 4 : 1;
  static constexpr int ROWS = 32 * RW;
  static constexpr int WKEYS = (WIDE ? ROW <= 512 : ROW <= 128) ? 64 : 32;  // keys of a stage that a wave works on
  static constexpr int STAGE = WIDE ? WKEYS : WKEYS * NW;
  static constexpr int BUFFER = STAGE * ROW;
  static constexpr int LDS = (WIDE ? 4 : 2) * BUFFER;      // K and V; where waves share them two buffers
  static constexpr int PER_CU = LDS <= 80 * 1024 ? 2 : 1;
  static constexpr int WGS = PA_CUS * PER_CU;
  static constexpr int WAVES = NW * PER_CU >= 4 ? NW * PER_CU / 4 : 1;  // per SIMD
  static constexpr int SLOT = ROWS * (DP + 2);             // floats of a part
  // 16-bit terms that a weight is taken apart into for the second product. Two where every wave has keys of its own: memory bounds that
  // form and the second term's products are free (64 single tokens, 779 us either way), the result is as exact as its own rounding (off
  // by 0.0017 in bf16, 0.0002 in fp16; with one term 0.0023 and 0.00026). One where waves share keys: matrix and vector instructions
  // bound it, and a second term takes 812 us instead of 639 (2048 tokens over 18432 keys) for the same gain. A weight is
  // off by half a step then, each by one of its own sign: on average less than the result's own rounding.
  static constexpr int TERMS = WIDE ? 1 : 2;
  // In keys: what starting and ending a tile takes (256: one request of 100 keys 17 us instead of 11, its 8 heads' tiles split), and
  // the least that is worth a workgroup (512: 5 fp32 requests of 2000 keys 43 us instead of 34; 128: no case gains, small ones lose 1).
  static constexpr int TILE_COST = 128;
  static constexpr int LEAST = 256;
  // A tile of this many keys or fewer is not split where a workgroup's piece is no more: its joining costs more than the longer work (16
  // requests under Sink + Local, 700 keys a tile: 36 -> 30 us, 2048 the same; 8 of one token and 200 keys: 18 -> 12). fp32, 16 times
  // the matrix time a key: 5 requests of 2000 keys 35 us, 38 with 256 or 384.
  static constexpr int WHOLE = DT == SAH_F32 ? 0 : WIDE ? 1024 : 512;
};

// The kernel's arguments where they lie. Each call gives an address that the compiler knows nothing of, so that what is read behind it is
// read again for every tile: all of them kept in scalar registers from the kernel's first line on, two hundred of those go
// to vector registers and come back in the innermost loop (2048 tokens over 18432 keys: 666 us instead of 647).
typedef const sah_paged_attention_args __attribute__((address_space(4))) pa_args;
__device__ __forceinline__ pa_args& pa_arguments() {
#if defined(__HIP_DEVICE_COMPILE__)
  pa_args* p = (pa_args*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
#else
  static pa_args* none;
  return *none;
#endif
}

// ---------------------------------------------------------------------------
// where the work is
// ---------------------------------------------------------------------------
struct pa_request {
  int row0, n_new;   // its rows of q
  int kv;            // keys it has
  int64_t base;      // row t stands at position base + t
};
__device__ __forceinline__ pa_request pa_read_request(pa_args& P, int b) {
  pa_request r;
  const int begin = P.cu_new[b], end = P.cu_new[b + 1];
  int kv = P.kv_lens[b];
  r.base = (int64_t)kv - end;
  r.row0 = begin < 0 ? 0 : (begin < P.n_tokens ? begin : P.n_tokens);
  const int e = end < P.n_tokens ? end : P.n_tokens;
  r.n_new = e > r.row0 ? e - r.row0 : 0;
  const int most = P.table_width * P.page_size;
  r.kv = kv < 0 ? 0 : (kv < most ? kv : most);
  return r;
}
// position of the request's i-th row, within what comparisons with key numbers need
__device__ __forceinline__ int pa_position(const pa_request& r, int i) {
  const int64_t p = r.base + r.row0 + i;
  return (int)(p < -1 ? -1 : (p < 0x7ffffffe ? p : 0x7ffffffe));
}

// What all lanes of the wave hold, in scalar registers (doubles are divided in vector ones)
__device__ __forceinline__ int64_t pa_uniform(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// a / b for 0 <= a < 2^53, 0 < b: exact. (The 64-bit division of integers is some 150 instructions, and a dozen of them stand
// before a workgroup's first load.)
__device__ __forceinline__ int64_t pa_div(int64_t a, int64_t b) {
  int64_t q = (int64_t)((double)a / (double)b);
  const int64_t r = a - q * b;
  q -= r < 0;
  q += r >= b;
  return q;
}

// Cost of the tiles of one request and head: tile i's is min(first + (i + 1) step, most) + each. About the keys it
// reads; only the balance depends on it.
struct pa_cost {
  int64_t first, step, most;
  int tiles, each;
  __device__ __forceinline__ int64_t of(int i) const {
    const int64_t c = first + (i + 1) * step;
    return (c < most ? c : most) + each;
  }
  __device__ __forceinline__ int64_t before(int i) const {  // of tiles 0 .. i - 1
    int64_t j = i;
    if (first + i * step > most) j = most > first ? pa_div(most - first, step) : 0;
    return j * first + step * (j * (j + 1) / 2) + (i - j) * most + (int64_t)i * each;
  }
  __device__ __forceinline__ int at(int64_t y) const {  // the tile whose piece of the line holds y
    int lo = 0, hi = tiles - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before(mid) <= y) lo = mid; else hi = mid - 1;
    }
    return lo;
  }
};
template <typename S>
__device__ __forceinline__ pa_cost pa_cost_of(pa_args& P, const pa_request& r) {
  const int G = P.Hq / P.Hkv;
  pa_cost c;
  c.each = S::TILE_COST;
  c.tiles = (int)(((int64_t)r.n_new * G + S::ROWS - 1) / S::ROWS);
  c.step = (S::ROWS + G - 1) / G;
  const int64_t p = r.base + r.row0;
  c.first = p < 0 ? 0 : (p < r.kv ? p : r.kv);
  c.most = P.window ? (int64_t)P.sink + P.window + c.step : (int64_t)1 << 40;
  return c;
}

// A place on the line of work: request, head, tile, and where the tile begins
struct pa_place {
  int b, hk, tile;
  int64_t begin, cost;
  pa_request req;
  pa_cost costs;
};

template <typename S>
__device__ __forceinline__ int pa_sharers(int64_t total) {
  const int64_t w = (total + S::LEAST - 1) / S::LEAST;
  return (int)(w < (int)gridDim.x ? w : (int)gridDim.x);
}
// This workgroup's number on the line of work: neighbours share keys, and parts of a tile, so they get the same XCD (the number of workgroups is a
// multiple of 8). The second kernel goes by the same numbers: by blockIdx.x itself the workgroups that begin a tile of 8 parts are all on
// one XCD, and read what others' L2s hold (62 us instead of 34 for 64 parts, 34 instead of 18 for 8).
__device__ __forceinline__ int pa_number() {
  return (int)(blockIdx.x % PA_XCDS) * (int)(gridDim.x / PA_XCDS) + (int)(blockIdx.x / PA_XCDS);
}
// where workgroup w of n begins
__device__ __forceinline__ int64_t pa_bound(int64_t total, int n, int w) {
  const int64_t each = pa_uniform(pa_div(total, n));
  return each * w + pa_uniform(pa_div((total - each * n) * w, n));
}

// The next tile on the line; there is one, unless lengths changed under way (an error of the program's, but one that ends)
template <typename S>
__device__ __forceinline__ bool pa_next(pa_args& P, pa_place& at) {
  at.begin += at.cost;
  if (++at.tile == at.costs.tiles) {
    at.tile = 0;
    if (++at.hk == P.Hkv) {
      at.hk = 0;
      do {
        if (++at.b >= P.n_requests) return false;
        at.req = pa_read_request(P, at.b);
        at.costs = pa_cost_of<S>(P, at.req);
      } while (at.costs.tiles == 0);
    }
  }
  at.cost = pa_uniform(at.costs.of(at.tile));
  return true;
}

// Workgroup w's piece of the line, [x0, x1), and the place that holds x0
struct pa_piece {
  int64_t total, x0, x1;
  int sharers;   // workgroups that have a piece; without one x0 and x1 say nothing
  int whole;     // tiles of at most this cost are one workgroup's, the one whose piece they begin in: x0 lies behind another's
  pa_place at;
  __device__ __forceinline__ bool none(int w) const { return w >= sharers || x0 >= x1; }
};
// s_sum: NT / 64 + 2 words. All NT threads call.
template <int NT, typename S>
__device__ __forceinline__ pa_piece pa_start(pa_args& P, int w, int64_t* s_sum) {
  constexpr int NW = NT / SAH_WAVE;
  const int lane = threadIdx.x % SAH_WAVE, wave = sah_wave_id();
  pa_piece r;
  auto cost_of = [&](int b) -> int64_t {
    if (b >= P.n_requests) return 0;
    const pa_cost c = pa_cost_of<S>(P, pa_read_request(P, b));
    return c.before(c.tiles) * P.Hkv;
  };
  auto scan = [&](int64_t v, int64_t& all) -> int64_t {  // inclusive
    const int64_t incl = (int64_t)sah_wave_incl_scan_u64((uint64_t)v);
    if (lane == SAH_WAVE - 1) s_sum[wave] = incl;
    __syncthreads();
    int64_t before = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      before += i < wave ? s_sum[i] : 0;
      all += s_sum[i];
    }
    all = pa_uniform(all);
    return before + incl;
  };
  auto share = [&](int64_t total) {
    r.total = total;
    r.sharers = pa_sharers<S>(total);
    r.x0 = w < r.sharers ? pa_bound(total, r.sharers, w) : 0;
    r.x1 = w < r.sharers ? pa_bound(total, r.sharers, w + 1) : 0;
  };
  auto claim = [&](int b, int64_t mine, int64_t end) {  // one thread's request holds x0
    if (mine && end > r.x0 && end - mine <= r.x0) {
      s_sum[NW] = b;
      s_sum[NW + 1] = end - mine;
    }
  };
  if (P.n_requests <= NT) {
    const int64_t mine = cost_of(threadIdx.x);
    int64_t all;
    const int64_t end = scan(mine, all);
    share(all);
    claim(threadIdx.x, mine, end);
    __syncthreads();
  } else {
    int64_t sum = 0, all, run = 0;
    for (int b = threadIdx.x; b < P.n_requests; b += NT) sum += cost_of(b);
    scan(sum, all);
    share(all);
    for (int b0 = 0; b0 < P.n_requests; b0 += NT) {
      const int64_t mine = cost_of(b0 + threadIdx.x);
      __syncthreads();
      const int64_t end = run + scan(mine, all);
      claim(b0 + threadIdx.x, mine, end);
      run += all;
    }
    __syncthreads();
  }
  if (w >= r.sharers) return r;
  pa_place& at = r.at;
  at.b = __builtin_amdgcn_readfirstlane((int)s_sum[NW]);
  const int64_t begin = pa_uniform(s_sum[NW + 1]);
  at.req = pa_read_request(P, at.b);
  at.costs = pa_cost_of<S>(P, at.req);
  const int64_t head = at.costs.before(at.costs.tiles);
  at.hk = (int)pa_uniform(pa_div(r.x0 - begin, head));
  at.tile = __builtin_amdgcn_readfirstlane(at.costs.at(r.x0 - begin - at.hk * head));
  at.begin = pa_uniform(begin + at.hk * head + at.costs.before(at.tile));
  at.cost = pa_uniform(at.costs.of(at.tile));
  r.whole = r.total <= (int64_t)S::WHOLE * r.sharers ? S::WHOLE : 0;
  if (r.x0 > at.begin && at.cost <= r.whole) {
    r.x0 = at.begin + at.cost;
    if (r.x0 < r.x1 && !pa_next<S>(P, at)) r.x0 = r.x1;
  }
  return r;
}

// what a workgroup leaves for the second kernel
struct pa_note {
  int b, hk, tile;  // the tile it began and others went on with; b < 0: none
  int last;         // the workgroup that ended it
  int again;        // some row of a whole tile came out not finite
  int pad[3];
};

// The stages that a tile's rows see: the first n_sink ones, then those from `from` on; `n` in all
struct pa_stages {
  int n, n_sink, from;
  __device__ __forceinline__ int operator()(int u) const { return u < n_sink ? u : u - n_sink + from; }
};
template <int STAGE>
__device__ __forceinline__ pa_stages pa_stages_of(pa_args& P, const pa_request& r, int p_lo, int p_hi) {
  pa_stages s;
  const int hi = p_hi < r.kv - 1 ? p_hi : r.kv - 1;  // the last key that any row sees
  s.n_sink = 0;
  s.from = 0;
  if (hi < 0) {
    s.n = 0;
    return s;
  }
  const int last = hi / STAGE;
  if (P.window) {
    const int first = p_lo >= P.window ? p_lo - P.window + 1 : 0;
    const int sink = P.sink < hi + 1 ? P.sink : hi + 1;
    const int sinks = (int)(((int64_t)sink + STAGE - 1) / STAGE);
    s.from = first / STAGE;
    if (sinks < s.from) {
      s.n_sink = sinks;
      s.n = sinks + (s.from <= last ? last - s.from + 1 : 0);
      return s;
    }
    s.from = 0;
  }
  s.n = last + 1;
  return s;
}

// How far a row's maximum may rise, in powers of two, before the row is rescaled (a rise of the maximum by a little is frequent,
// by 2^SLACK rare), and the power of two that the weights are held above their true size by: they enter the second product in
// terms of the tensor's type, and fp16 keeps all its bits for weights down to 2^-22 of the row's largest that way.
template <int DT> struct pa_weights {
  static constexpr float SLACK = DT == SAH_F16 ? 6.0f : 8.0f;
  static constexpr float SCALE = DT == SAH_F16 ? 8.0f : 0.0f;
};

// Results from here on (or NaN) are done again: the type has no finite number for them, while the average of finite values is one. (Weights
// of one term each half a step too large reach this where all values are the type's largest.)
template <int DT>
__device__ __forceinline__ bool pa_fine(float v) { return fabsf(v) < (DT == SAH_F32 ? INFINITY : DT == SAH_BF16 ? 0x1.ffp127f : 65520.f); }

// Reads of LDS written above this are issued above it, and x, the result of an earlier one, is used below it alone. (Left to itself the
// compiler reads where it multiplies, one wait of LDS's latency after the other.)
__device__ __forceinline__ void pa_reads_stay() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" ::: "memory");
#endif
}
__device__ __forceinline__ void pa_from_here(sah_u4& x) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(x)::"memory");
#endif
}
__device__ __forceinline__ uint4 pa_operand(const sah_u4& v) { return make_uint4(v.x, v.y, v.z, v.w); }

// Waits until no more than N of this wave's loads (LDS: 15 is no wait) are under way. The builtin, not an instruction of inline asm: the
// compiler counts loads itself, and where it does not see that staged keys have landed it waits for all loads there are.
template <int LOADS, int LDS>
__device__ __forceinline__ void pa_wait() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LOADS & 15) | 7 << 4 | LDS << 8 | (LOADS >> 4) << 14);
  asm volatile("" ::: "memory");
#endif
}
template <int N>
__device__ __forceinline__ void pa_landed() { pa_wait<N, 15>(); }
// What this wave has asked LDS for has been read.
__device__ __forceinline__ void pa_lds_read() { pa_wait<63, 0>(); }

template <int DT, int DP, bool WIDE>
__global__ __launch_bounds__((pa_shape<DT, DP, WIDE>::NT), (pa_shape<DT, DP, WIDE>::WAVES)) void k_paged_attn(sah_paged_attention_args) {
  sah_touch_kernargs<sizeof(sah_paged_attention_args)>();
  typedef pa_shape<DT, DP, WIDE> S;
  constexpr int ES = S::ES, NT = S::NT, UNITS = S::ROW / 16;
  constexpr int KPI = SAH_WAVE / (UNITS < 64 ? UNITS : 64);    // keys per load instruction
  constexpr int IW = S::WKEYS / KPI / (WIDE ? S::NW : 1);      // load instructions per wave, matrix and stage
  constexpr int IG = 16 / KPI < IW ? 16 / KPI : IW;            // ... of them that are 16 keys (or all)
  constexpr int TW = S::WKEYS / 32;                            // 32-key tiles a wave works on in a stage
  constexpr int DTL = DP / 32;
  constexpr int KQ = DT == SAH_F32 ? DP / 8 : DP / 16;         // 16-byte pieces of a lane's query
  static_assert(UNITS <= 64 && IW >= 1, "a key is at most one load instruction");
  // K and V as they lie in memory, a row per key, its 16-byte units permuted against bank conflicts: K unit c of key j at
  // place c ^ (j % 16) (8 units: c ^ (j / 2 % 8)); V of 16-bit types: groups of four units (32 dims) at place
  // u ^ (j % 4) (8 units: u ^ (j / 2 % 2)) for the transposing reads. (An array each: the compiler then knows that what is
  // read is not what the loads under way will write.)
  constexpr int SB = S::BUFFER, SB1 = WIDE ? SB : 16;
  __shared__ __align__(16) unsigned char s_k0[SB], s_k1[SB1], s_v0[SB], s_v1[SB1];
  __shared__ int64_t s_sum[S::NW + 2];
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const int i32 = lane & 31, g = lane >> 5;
  const int rw = WIDE ? wave : 0;
  const int w = pa_number();
  if (threadIdx.x == 0) {
    pa_note* note = (pa_note*)pa_arguments().work + w;
    note->b = -1;
    note->again = 0;
  }
  const pa_piece piece = pa_start<NT, S>(pa_arguments(), w, s_sum);
  const int sharers = piece.sharers;
  if (piece.none(w)) return;
  const int64_t total = piece.total, x1 = piece.x1;
  int64_t x = piece.x0;
  pa_place at = piece.at;
  // this lane's share of a load instruction, and where it reads what has been staged
  const int l_key = lane / UNITS, l_place = lane % UNITS;
  auto f_k = [](int key) { return UNITS == 8 ? (key >> 1) & 7 : key & 15; };
  auto f_v = [](int key) { return DT == SAH_F32 ? 0 : UNITS == 8 ? 4 * ((key >> 1) & 1) : 4 * (key & 3); };
  const int k_at = i32 * S::ROW + 16 * (g ^ f_k(i32));
  int v_at[DTL];
#pragma unroll
  for (int t = 0; t < DTL; ++t) {
    const int row = 4 * g + ((lane & 15) >> 2);
    v_at[t] = row * S::ROW + 16 * ((4 * t) ^ f_v(row)) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  }

  bool bad = false;  // a row of a whole tile came out not finite
  for (;;) {
    pa_args& P = pa_arguments();
    const int G = P.Hq / P.Hkv, page_shift = 31 - __builtin_clz(P.page_size);
    const float c_exp = fmaxf(fabsf(P.scaling) * 1.4426950408889634f, 1e-37f);
    // (places behind a shorter head's end hold its last unit again: the queries are 0 there, the results nobody's)
    const int units_real = P.D * ES / 16;
    const uint32_t last_unit = 16u * (units_real - 1);
    const uint32_t k_unit = 16u * (l_place ^ f_k(l_key)), v_unit = 16u * (l_place ^ f_v(l_key));
    // an instruction's keys lie in one page, and a key's elements before the next key's
    const bool regular = P.page_size >= KPI && P.ks_t >= P.D && P.vs_t >= P.D;
    const uint32_t k_step = (uint32_t)(KPI * P.ks_t * ES), v_step = (uint32_t)(KPI * P.vs_t * ES);  // from an instruction's keys to the next one's
    const uint32_t k_lane = (uint32_t)(l_key * P.ks_t * ES), v_lane = (uint32_t)(l_key * P.vs_t * ES);
    const int64_t y0 = x - at.begin, y1 = x1 - at.begin < at.cost && at.cost > piece.whole ? x1 - at.begin : at.cost;
    const bool whole = y0 == 0 && y1 == at.cost;
    const int row_first = at.tile * S::ROWS;
    const int n_rows = at.req.n_new * G;  // (n_new <= n_tokens, and n_tokens * Hq fits: the host has checked)
    const int row_last = row_first + S::ROWS < n_rows ? row_first + S::ROWS - 1 : n_rows - 1;
    const pa_stages stages = pa_stages_of<S::STAGE>(P, at.req, pa_position(at.req, row_first / G), pa_position(at.req, row_last / G));
    const int u0 = y0 == 0 ? 0 : (int)pa_uniform(pa_div(y0 * stages.n, at.cost)), u1 = y1 == at.cost ? stages.n : (int)pa_uniform(pa_div(y1 * stages.n, at.cost));

    // this lane's rows; lanes beyond the last repeat it and store nothing
    // (its place in the wave is taken anew for every tile, as the kernel's arguments are: what follows from it, kept, is 80 registers)
    uint32_t kept_lane = lane;
    sah_keep(kept_lane);
    const int i32 = kept_lane & 31, g = kept_lane >> 5;
    int pos, tok, head;
    bool live;
    uint4 qf[KQ];
    bool wave_live = false;
    int w_lo = 0x7fffffff, w_hi = -1;  // positions of the wave's rows
    const int r0 = row_first + rw * 32;
    if (r0 < n_rows) {
      wave_live = true;
      const int r1 = r0 + 31 < n_rows ? r0 + 31 : n_rows - 1;
      const int a = pa_position(at.req, r0 / G), z = pa_position(at.req, r1 / G);
      w_lo = a < w_lo ? a : w_lo;
      w_hi = z > w_hi ? z : w_hi;
    }
    const int r = r0 + i32;
    live = r < n_rows;
    const int rr = live ? r : n_rows - 1;
    const int i = rr / G;
    head = at.hk * G + rr - i * G;
    tok = at.req.row0 + i;
    pos = pa_position(at.req, i);
    const char* qp = (const char*)P.q + ((int64_t)tok * P.qs_t + (int64_t)head * P.qs_h) * ES;
#pragma unroll
    for (int s = 0; s < KQ; ++s) {
      const int unit = 2 * s + g;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (unit < units_real) v = *(const uint4*)(qp + 16 * unit);
      if (P.scaling < 0.f) {  // uniform: the sign is the query's
        const uint32_t sign = DT == SAH_F32 ? 0x80000000u : 0x80008000u;
        v.x ^= sign; v.y ^= sign; v.z ^= sign; v.w ^= sign;
      }
      qf[s] = v;
    }
    w_lo = __builtin_amdgcn_readfirstlane(w_lo);
    w_hi = __builtin_amdgcn_readfirstlane(w_hi);

    float m_run, l_run;
    sah_f32x16 acc[DTL];
    m_run = -INFINITY;
    l_run = 0.f;
#pragma unroll
    for (int t = 0; t < DTL; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[t][e] = 0.f;

    // The keys of a stage that this wave works on: a lane holds the page of one, and a bit says which are there. Requested a
    // stage ahead of the loads that go by it.
    const int32_t* table = P.block_table + (int64_t)at.b * P.table_pitch;
    [[maybe_unused]] int page = -1, page_next = -1;
    auto first_key = [&](int u) { return stages(u) * S::STAGE + (WIDE ? 0 : S::WKEYS * wave); };
    auto fetch_page = [&](int u) -> int {
      const int key = first_key(u) + (S::WKEYS == 64 ? lane : i32);
      return key < at.req.kv ? table[key >> page_shift] : -1;
    };
    auto there_of = [&](int pg) -> uint64_t {
      const uint64_t m = __ballot(pg >= 0 && pg < P.n_pages);
      return S::WKEYS == 64 ? m : m & 0xffffffffu;
    };
    const char* kbase = (const char*)P.k + (int64_t)at.hk * P.ks_h * ES;
    const char* vbase = (const char*)P.v + (int64_t)at.hk * P.vs_h * ES;
    auto fetch = [&](int u, int pg, uint64_t there, int buf, bool with_k, bool with_v) __attribute__((always_inline)) {
      const int key0 = first_key(u);
      auto stage_at = [&](int at_key) { return ((WIDE ? 0 : S::WKEYS * wave) + at_key) * S::ROW; };
      const int left = at.req.kv - key0;  // the request's keys from here on
      const uint64_t held = left >= S::WKEYS ? (S::WKEYS == 64 ? ~0ull : 0xffffffffull) : left > 0 ? (1ull << left) - 1 : 0;
      // All of them are there and the keys of GI instructions lie in one page: a scalar base for these, and lanes' offsets that stay
      // the same (the permutation's part of an instruction is an exclusive or: its key's bits are none of the lane's, and the
      // groups' begin with 16 keys). Keys behind the request's last come as zeros.
      auto fast = [&](auto group) __attribute__((always_inline)) {
        constexpr int GI = decltype(group)::value;
#pragma unroll
        for (int i0 = 0; i0 < IW; i0 += GI) {
          const int first = ((WIDE ? wave * IW : 0) + i0) * KPI;
          const int here = left - first, page_of = __builtin_amdgcn_readlane(pg, first);
          const int64_t p = here > 0 ? page_of : 0, entry = (key0 + first) & (P.page_size - 1);
          const char* ka = kbase + (p * P.ks_p + entry * P.ks_t) * ES;
          const char* va = vbase + (p * P.vs_p + entry * P.vs_t) * ES;
          const uint32_t k_bytes = here >= GI * KPI ? ~0u : here > 0 ? (uint32_t)(here * P.ks_t * ES) : 0u;
          const uint32_t v_bytes = here >= GI * KPI ? ~0u : here > 0 ? (uint32_t)(here * P.vs_t * ES) : 0u;
#pragma unroll
          for (int i = 0; i < GI; ++i) {
            const int at_key = first + i * KPI, turn = GI == IG ? i * KPI : at_key;
            const uint32_t uk = k_unit ^ (16u * f_k(turn)), uv = v_unit ^ (16u * f_v(turn));
            if (with_k) sah_buffer_load_lds16(ka, k_bytes, k_lane + i * k_step + (uk < last_unit ? uk : last_unit), (buf ? s_k1 : s_k0) + stage_at(at_key));
            if (with_v) sah_buffer_load_lds16(va, v_bytes, v_lane + i * v_step + (uv < last_unit ? uv : last_unit), (buf ? s_v1 : s_v0) + stage_at(at_key));
          }
        }
      };
      if (there == held && regular) {  // uniform
        if (P.page_size >= 16) fast(std::integral_constant<int, IG>());
        else fast(std::integral_constant<int, 1>());
        return;
      }
      // Keys that are not there, or pages smaller than an instruction's keys: every lane its own address, through registers. (A
      // stage's K and V both come this way or neither: the count of loads under way holds.)
      const int spare = 63 - __builtin_clzll(there | 1);  // stands for keys that are not there
      constexpr int U = IW < 2 ? IW : 2;
#pragma unroll 1
      for (int i0 = 0; i0 < IW; i0 += U) {
        sah_u4 k[U], v[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int key = ((WIDE ? wave * IW : 0) + i0 + i) * KPI + l_key;
          const int src = (there >> key) & 1 ? key : spare;
          const int page_of = __shfl(pg, src);
          const int64_t p = there ? page_of : 0;  // (nothing there: any page, and nobody reads it)
          const int64_t entry = (key0 + src) & (P.page_size - 1);
          const uint32_t uk = 16u * (l_place ^ f_k(key)), uv = 16u * (l_place ^ f_v(key));
          if (with_k) k[i] = *(const sah_u4*)(kbase + (p * P.ks_p + entry * P.ks_t) * ES + (uk < last_unit ? uk : last_unit));
          if (with_v) v[i] = *(const sah_u4*)(vbase + (p * P.vs_p + entry * P.vs_t) * ES + (uv < last_unit ? uv : last_unit));
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int to = stage_at(((WIDE ? wave * IW : 0) + i0 + i) * KPI) + 16 * lane;
          if (with_k) *(sah_u4*)((buf ? s_k1 : s_k0) + to) = k[i];
          if (with_v) *(sah_u4*)((buf ? s_v1 : s_v0) + to) = v[i];
        }
      }
    };

    // `between` runs when the stage's keys have been read, before its values are
    auto work = [&](int u, uint64_t there, int buf, auto between) __attribute__((always_inline)) {
      const int key0 = first_key(u);
      const bool on = wave_live && there != 0 && key0 <= w_hi;  // uniform
      const unsigned char* kp = (buf ? s_k1 : s_k0) + (WIDE ? 0 : S::WKEYS * wave * S::ROW);
      const unsigned char* vp = (buf ? s_v1 : s_v0) + (WIDE ? 0 : S::WKEYS * wave * S::ROW);
      sah_f32x16 s[TW];
#pragma unroll
      for (int t = 0; t < TW; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
      // PA_LOOK pieces of a key tile at a time are read while as many before are multiplied.
      if (on) {
        __builtin_amdgcn_s_setprio(1);  // while one wave of a SIMD multiplies another finds its softmax's turns by itself
        constexpr int C = PA_LOOK, NC = TW * KQ / C;
        sah_u4 a[2][C];
        auto read = [&](int c) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < C; ++i) {
            const int t = c * C / KQ, st = c * C % KQ + i;
            a[c & 1][i] = *(const sah_u4*)(kp + 32 * t * S::ROW + (k_at ^ (32 * st)));
          }
        };
        read(0);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (c + 1 < NC) read(c + 1);
#pragma unroll
          for (int i = 0; i < C; ++i) pa_from_here(a[c & 1][i]);
#pragma unroll
          for (int i = 0; i < C; ++i) {
            const int t = c * C / KQ, st = c * C % KQ + i;
            const uint4 k = pa_operand(a[c & 1][i]);
            if constexpr (DT == SAH_F32) {
              s[t] = sah_mfma_32x32x2_f32(sah_bits_to_float(k.x), sah_bits_to_float(qf[st].x), s[t]);
              s[t] = sah_mfma_32x32x2_f32(sah_bits_to_float(k.y), sah_bits_to_float(qf[st].y), s[t]);
              s[t] = sah_mfma_32x32x2_f32(sah_bits_to_float(k.z), sah_bits_to_float(qf[st].z), s[t]);
              s[t] = sah_mfma_32x32x2_f32(sah_bits_to_float(k.w), sah_bits_to_float(qf[st].w), s[t]);
            } else {
              s[t] = sah_mfma_32x32x16<DT>(k, qf[st], s[t]);
            }
          }
        }
      }
      __builtin_amdgcn_s_setprio(0);
      between();
      if (!on) return;
      // the first values, requested ahead of the softmax
      constexpr int DV = DTL < PA_LOOK_V ? DTL : PA_LOOK_V, NV = 2 * TW * (DTL / DV);  // 32-dim tiles of a piece, pieces
      sah_u4 va[2][DT == SAH_F32 ? 1 : DV];
      auto read_v = [&](int c) __attribute__((always_inline)) {
        if constexpr (DT != SAH_F32) {
#pragma unroll
          for (int d = 0; d < DV; ++d) {
            const unsigned char* v = vp + 16 * (c / (DTL / DV)) * S::ROW + v_at[c % (DTL / DV) * DV + d];
            const sah_u2 a0 = sah_read_tr16((const uint16_t*)v), a1 = sah_read_tr16((const uint16_t*)(v + 8 * S::ROW));
            va[c & 1][d] = sah_u4{a0.x, a0.y, a1.x, a1.y};
          }
        }
      };
      read_v(0);
      pa_reads_stay();
      // every row sees every key of the stage?
      const uint64_t full = S::WKEYS == 64 ? ~0ull : 0xffffffffull;
      const bool plain = there == full && key0 + S::WKEYS - 1 <= w_lo &&
                         (!P.window || key0 + S::WKEYS <= P.sink || (int64_t)key0 > (int64_t)w_hi - P.window);
      if (!plain) {
        uint32_t kept_pos = pos;
        sah_keep(kept_pos);
        const int at_pos = (int)kept_pos;
        const int lo = P.window && at_pos >= P.window ? at_pos - P.window + 1 : 0;
#pragma unroll
        for (int t = 0; t < TW; ++t) {
          const int k0 = key0 + 32 * t, wi = k0 / 32;
          uint32_t word = sah_range_bits(wi, lo, at_pos + 1);
          if (P.window) word |= sah_range_bits(wi, 0, P.sink < at_pos + 1 ? P.sink : at_pos + 1);
          word &= (uint32_t)(there >> (32 * t));
          word >>= 4 * g;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint32_t on = (uint32_t)((int)(word << (31 - (8 * (e / 4) + e % 4))) >> 31);  // all ones where the row sees the key
            s[t][e] = sah_bits_to_float((sah_float_to_bits(s[t][e]) & on) | (0xff800000u & ~on));
          }
        }
      }
      float mc;
      float mx = s[0][0];
#pragma unroll
      for (int t = 0; t < TW; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
      mx = sah_half_max(mx) * c_exp;
      // (-inf - -inf is NaN: no rise)
      if (__ballot(mx - m_run > pa_weights<DT>::SLACK) != 0) {  // uniform: some row's maximum has risen too far
        const float m_new = fmaxf(m_run, mx);
        const float up = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= up;
#pragma unroll
        for (int t = 0; t < DTL; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[t][e] *= up;
      }
      // (a row that has seen nothing: in range, so that -inf comes to 0)
      mc = (m_run == -INFINITY ? 0.f : m_run) - pa_weights<DT>::SCALE;
      auto weigh = [&](int t, int e0, int n) __attribute__((always_inline)) {  // n of a key tile's weights
#pragma unroll
          for (int e = e0; e < e0 + n; ++e) {
            s[t][e] = __builtin_amdgcn_exp2f(fmaf(s[t][e], c_exp, -mc));
            l_run += s[t][e];
          }
      };
      // (16-bit types: the second key tile's weights are taken between the first one's products)
#pragma unroll
      for (int t = 0; t < (DT == SAH_F32 ? TW : 1); ++t) weigh(t, 0, 16);
      if constexpr (DT == SAH_F32) {
#pragma unroll
        for (int t = 0; t < TW; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float* row = (const float*)(vp + (32 * t + 8 * (e / 4) + e % 4 + 4 * g) * S::ROW) + i32;
#pragma unroll
            for (int d = 0; d < DTL; ++d) {
              const float v = row[32 * d];
              acc[d] = sah_mfma_32x32x2_f32(v, s[t][e], acc[d]);
            }
          }
      } else {
        __builtin_amdgcn_s_setprio(1);
        uint32_t term[S::TERMS][4];
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          const int step = c / (DTL / DV), t = step / 2, st = step % 2;
          if (c + 1 < NV) read_v(c + 1);
#pragma unroll
          for (int d = 0; d < DV; ++d) pa_from_here(va[c & 1][d]);
          const auto& z = s[t];
          if (c % (DTL / DV) == 0) {  // the step's weights: as they are rounded, and what the rounding has cut off
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              float p0 = z[8 * st + 2 * p], p1 = z[8 * st + 2 * p + 1];
#pragma unroll
              for (int i = 0; i < S::TERMS; ++i) {
                term[i][p] = sah_pack2_hw<DT>(p0, p1);
                if (i + 1 == S::TERMS) break;
                sah_keep(term[i][p]);  // taken apart as it is, instead of converted a second time
                if (DT == SAH_BF16) {
                  p0 -= sah_bits_to_float(term[i][p] << 16);
                  p1 -= sah_bits_to_float(term[i][p] & 0xffff0000u);
                } else {
                  p0 -= sah_f16_to_float((uint16_t)term[i][p]);
                  p1 -= sah_f16_to_float((uint16_t)(term[i][p] >> 16));
                }
              }
            }
          }
#pragma unroll
          for (int i = 0; i < S::TERMS; ++i)
#pragma unroll
            for (int d = 0; d < DV; ++d) {
              const int to = c % (DTL / DV) * DV + d;
              acc[to] = sah_mfma_32x32x16<DT>(pa_operand(va[c & 1][d]), make_uint4(term[i][0], term[i][1], term[i][2], term[i][3]), acc[to]);
            }
          if (TW == 2 && t == 0) {
            constexpr int N = 16 * TW / NV;
            weigh(1, c * N, N);
          }
        }
        __builtin_amdgcn_s_setprio(0);
      }
    };

    if constexpr (WIDE) {
      auto stage = [&](int u, int buf) __attribute__((always_inline)) {  // buf: a constant in the loop below
        const uint64_t there = there_of(page);
        if (u + 1 < u1) {
          page = page_next;
          fetch(u + 1, page, there_of(page), buf ^ 1, true, true);  // the other buffer: read for the last time before the previous wait
          if (u + 2 < u1) page_next = fetch_page(u + 2);
        }
        work(u, there, buf, [] {});
        sah_stores_done();  // this wave's loads into LDS have landed
        __syncthreads();
      };
      if (u0 < u1) {
        page = fetch_page(u0);
        if (u0 + 1 < u1) page_next = fetch_page(u0 + 1);
        fetch(u0, page, there_of(page), 0, true, true);
        sah_stores_done();
        __syncthreads();
        for (int u = u0; u < u1; u += 2) {
          stage(u, 0);
          if (u + 1 < u1) stage(u + 1, 1);
        }
      }
    } else {
      // A wave's own keys, with nobody to wait for: a stage's K is overwritten by the next one's as soon as it has been multiplied,
      // its V likewise, so that half a stage of loads or more is under way all the time (8 waves of 16 KB a stage and CU at 128 x 2
      // bytes). Loads land in the order they were asked for in: waiting for K means waiting until no more than what was
      // requested after it is left. Pages are requested a stage ahead of the loads that go by them.
      static_assert(IW <= 32, "counted in six bits");
      if (u0 < u1) {
        int pg = fetch_page(u0);
        int pg_next = u0 + 1 < u1 ? fetch_page(u0 + 1) : -1;
        uint64_t there = there_of(pg);
        fetch(u0, pg, there, 0, true, false);
        fetch(u0, pg, there, 0, false, true);
        // (the last stage apart: a way through the loop that skips a request would have the compiler wait for all of them)
        int u = u0;
#pragma unroll 1
        for (; u + 1 < u1; ++u) {
          uint64_t there_next = 0;
          pa_landed<IW>();  // K
          work(u, there, 0, [&]() __attribute__((always_inline)) {
            pg = pg_next;
            there_next = there_of(pg);
            pg_next = fetch_page(u + 2 < u1 ? u + 2 : u + 1);
            pa_lds_read();
            fetch(u + 1, pg, there_next, 0, true, false);
            pa_landed<IW>();  // V
          });
          pa_lds_read();
          fetch(u + 1, pg, there_next, 0, false, true);
          there = there_next;
        }
        pa_landed<IW>();
        work(u, there, 0, []() __attribute__((always_inline)) { pa_landed<0>(); });
        pa_landed<0>();
      }
    }

    l_run = sah_half_sum(l_run);
    // A lane holds 4 * DTL groups of four neighbouring dims of its row. Where every wave had keys of its own, all waves' are added up in
    // LDS, each wave taking a share of the groups (one wave doing it for all: 6.5 us of a part's end).
    constexpr int GROUPS = 4 * DTL, MINE = WIDE ? GROUPS : GROUPS / S::NW;
    [[maybe_unused]] float up[S::NW];
    if constexpr (!WIDE && S::NW > 1) {
      __shared__ float s_ml[S::NW][2][SAH_WAVE];
      constexpr int PER = SB / (GROUPS * SAH_WAVE * 16);  // waves that a buffer holds, [group][lane]
      static_assert(PER >= 1 && PER * 2 >= S::NW && MINE * S::NW == GROUPS, "room for the waves' shares");
      __syncthreads();  // every wave has read its stages
      float4* to = (float4*)(wave < PER ? s_k0 : s_v0) + wave % PER * GROUPS * SAH_WAVE + lane;
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        const auto& v = acc[i / 4];
        to[i * SAH_WAVE] = make_float4(v[4 * (i % 4)], v[4 * (i % 4) + 1], v[4 * (i % 4) + 2], v[4 * (i % 4) + 3]);
      }
      s_ml[wave][0][lane] = m_run;
      s_ml[wave][1][lane] = l_run;
      __syncthreads();
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int v = 0; v < S::NW; ++v) m = fmaxf(m, s_ml[v][0][lane]);
#pragma unroll
      for (int v = 0; v < S::NW; ++v) {
        const float mv = s_ml[v][0][lane];
        up[v] = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mv - m);
        l += s_ml[v][1][lane] * up[v];
      }
      m_run = m;
      l_run = l;
    }
    // group i of this wave's, its number among all
    auto group_of = [&](int i, int& number) __attribute__((always_inline)) -> float4 {
      if constexpr (!WIDE && S::NW > 1) {
        constexpr int PER = SB / (GROUPS * SAH_WAVE * 16);
        number = wave * MINE + i;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int v = 0; v < S::NW; ++v) {
          const float4 a = ((const float4*)(v < PER ? s_k0 : s_v0))[(v % PER * GROUPS + number) * SAH_WAVE + lane];
          sum.x += a.x * up[v];
          sum.y += a.y * up[v];
          sum.z += a.z * up[v];
          sum.w += a.w * up[v];
        }
        return sum;
      } else {
        number = i;
        const auto& v = acc[i / 4];
        return make_float4(v[4 * (i % 4)], v[4 * (i % 4) + 1], v[4 * (i % 4) + 2], v[4 * (i % 4) + 3]);
      }
    };
    {
      pa_args& P = pa_arguments();
      uint32_t kept_again = lane;
      sah_keep(kept_again);
      const int i32 = kept_again & 31, g = kept_again >> 5;
      if (whole) {
        float l = l_run;
        if (P.sinks) {
          // a row that has seen nothing has nothing to weigh against its sink
          const float z = fmaf(P.sinks[head], 1.4426950408889634f, pa_weights<DT>::SCALE) - m_run;
          if (m_run != -INFINITY) l += __builtin_amdgcn_exp2f(z);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bool fine = true;
        char* op = (char*)P.out + ((int64_t)tok * P.os_t + (int64_t)head * P.os_h) * ES;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          int number;
          const float4 a = group_of(i, number);
          const int d = 8 * number + 4 * g;
          if (d >= P.D) continue;
          const float4 o = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
          fine = fine && pa_fine<DT>(o.x) && pa_fine<DT>(o.y) && pa_fine<DT>(o.z) && pa_fine<DT>(o.w);
          if (!live) continue;
          if (DT == SAH_F32) *(float4*)(op + 4 * d) = o;
          else *(uint2*)(op + 2 * d) = make_uint2(sah_pack2_hw<DT>(o.x, o.y), sah_pack2_hw<DT>(o.z, o.w));
        }
        bad = bad || (live && !fine);
      } else {
        // a part: to slot 0 where the tile began before this workgroup's piece, else to slot 1
        float* to = P.work + S::WGS * (sizeof(pa_note) / 4) + (int64_t)(2 * w + (y0 ? 0 : 1)) * S::SLOT;
        const int r = rw * 32 + i32;
        if (live && g == 0 && (WIDE || wave == 0)) ((float2*)to)[r] = make_float2(m_run, l_run);
        float* o = to + 2 * S::ROWS + r * DP;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          int number;
          const float4 a = group_of(i, number);
          if (live) *(float4*)(o + 8 * number + 4 * g) = a;
        }
        if (y0 == 0 && threadIdx.x == 0) {
          // the workgroup whose piece holds the tile's last key: the first whose end is not before the tile's
          const int64_t end = at.begin + at.cost;
          int last = (int)((double)end / (double)total * sharers);
          last = last < sharers ? last : sharers - 1;
          while (last + 1 < sharers && pa_bound(total, sharers, last + 1) < end) ++last;
          while (last > w && pa_bound(total, sharers, last) >= end) --last;
          pa_note* note = (pa_note*)P.work + w;
          note->hk = at.hk;
          note->tile = at.tile;
          note->last = last;
          note->b = at.b;
        }
      }
    }
    x = at.begin + y1;
    if (x >= x1) break;
    if (!WIDE) __syncthreads();  // all shares have been read
    if (!pa_next<S>(pa_arguments(), at)) break;
  }
  if (bad) ((pa_note*)pa_arguments().work)[w].again = 1;
}

// One row key by key, by one wave: what a row holds whose products in a tile came out not finite. The average so far is held, not the
// sum: of finite values it is finite, however large they are.
template <int DT>
__device__ __forceinline__ void pa_row_again(pa_args& P, const pa_request& r, int b, int t, int h) {
  constexpr int E = PA_MAX_D / SAH_WAVE;
  const int lane = threadIdx.x & (SAH_WAVE - 1), hk = h / (P.Hq / P.Hkv);
  const int64_t p = r.base + t;
  const int64_t end = p + 1 < r.kv ? p + 1 : r.kv;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + e * SAH_WAVE;
    q[e] = d < P.D ? sah_load<DT>(P.q, (int64_t)t * P.qs_t + (int64_t)h * P.qs_h + d) : 0.f;
    acc[e] = 0.f;
  }
  for (int64_t j = 0; j < end; ++j) {
    if (P.window > 0 && j >= P.sink && j <= p - P.window) continue;
    const int page = P.block_table[(int64_t)b * P.table_pitch + j / P.page_size];
    if (page < 0 || page >= P.n_pages) continue;
    const int64_t in = j % P.page_size;
    const int64_t ka = page * P.ks_p + in * P.ks_t + hk * P.ks_h, va = page * P.vs_p + in * P.vs_t + hk * P.vs_h;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + e * SAH_WAVE;
      if (d < P.D) s = fmaf(q[e], sah_load<DT>(P.k, ka + d), s);
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
      if (d < P.D) acc[e] = acc[e] * old + share * sah_load<DT>(P.v, va + d);
    }
  }
  const float seen = P.sinks && m != -INFINITY ? l / (l + expf(P.sinks[h] - m)) : 1.f;  // all but the sink's share
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + e * SAH_WAVE;
    if (d < P.D) sah_store<DT>(P.out, (int64_t)t * P.os_t + (int64_t)h * P.os_h + d, acc[e] * seen);
  }
}

// Joins the parts of the tile that this workgroup's number in the first kernel began and did not end. 16 lanes hold a row: with few parts
// a workgroup does 16 rows at once, with many one row, whose parts its 16 groups take in turn. blockIdx.y shares the rows out.
#define PA_JOIN_NT 256
#define PA_JOIN_GROUPS (PA_JOIN_NT / 16)
#define PA_JOIN_WGS 8
template <int DT, int DP, bool WIDE>
__global__ __launch_bounds__(PA_JOIN_NT) void k_paged_attn_join(sah_paged_attention_args) {
  sah_touch_kernargs<sizeof(sah_paged_attention_args)>();
  pa_args& P = pa_arguments();
  typedef pa_shape<DT, DP, WIDE> S;
  constexpr int NW = PA_JOIN_NT / SAH_WAVE, F = DP / 64;  // float4s of a lane: dims 4 (lane % 16) + 64 f ..
  __shared__ float s_ml[PA_JOIN_GROUPS][2];
  __shared__ float4 s_acc[PA_JOIN_GROUPS][DP / 4];
  __shared__ int64_t s_sum[NW + 2];
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const int group = threadIdx.x / 16, l16 = threadIdx.x % 16;
  const int w = pa_number(), G = P.Hq / P.Hkv;
  const pa_note note = ((const pa_note*)P.work)[w];
  const float* parts = P.work + S::WGS * (sizeof(pa_note) / 4);
  if (note.b >= 0) {
    const pa_request req = pa_read_request(P, note.b);
    const int n_rows = req.n_new * G - note.tile * S::ROWS < S::ROWS ? req.n_new * G - note.tile * S::ROWS : S::ROWS;
    const int n_parts = note.last - w + 1;
    // whichever has fewer trips to memory in a row
    const bool many = (n_parts + 3) / 4 * ((n_rows + PA_JOIN_WGS * PA_JOIN_GROUPS - 1) / (PA_JOIN_WGS * PA_JOIN_GROUPS)) >
                      (n_rows + PA_JOIN_WGS - 1) / PA_JOIN_WGS * (n_parts / (4 * PA_JOIN_GROUPS) + 2);
    for (int i0 = blockIdx.y * (many ? 1 : PA_JOIN_GROUPS); i0 < n_rows; i0 += PA_JOIN_WGS * (many ? 1 : PA_JOIN_GROUPS)) {  // uniform
      const int i = many ? i0 : i0 + group < n_rows ? i0 + group : n_rows - 1;
      const int first = many ? group : 0, step = many ? PA_JOIN_GROUPS : 1;
      float m = -INFINITY, l = 0.f;
      float4 acc[F];
#pragma unroll
      for (int f = 0; f < F; ++f) acc[f] = make_float4(0.f, 0.f, 0.f, 0.f);
      auto add = [&](float2 ml, const float4 (&v)[F]) __attribute__((always_inline)) {
        const float m_new = fmaxf(m, ml.x);
        const float a = m == -INFINITY ? 0.f : exp2f(m - m_new), z = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m_new);
        // (a part whose sum is NaN has no maximum, perhaps: the row is done again all the same)
        l = l * a + (ml.y == ml.y ? ml.y * z : ml.y);
        m = m_new;
#pragma unroll
        for (int f = 0; f < F; ++f) {
          acc[f].x = acc[f].x * a + v[f].x * z;
          acc[f].y = acc[f].y * a + v[f].y * z;
          acc[f].z = acc[f].z * a + v[f].z * z;
          acc[f].w = acc[f].w * a + v[f].w * z;
        }
      };
      constexpr int U = 4;
      for (int p = first; p < n_parts; p += U * step) {  // four parts requested at once; behind the last one it is taken again, and not added
        float2 ml[U];
        float4 v[U][F];
#pragma unroll
        for (int q = 0; q < U; ++q) {
          const int pp = p + q * step < n_parts ? p + q * step : n_parts - 1;
          const float* from = parts + (int64_t)(pp ? 2 * (w + pp) : 2 * w + 1) * S::SLOT;
          ml[q] = ((const float2*)from)[i];
#pragma unroll
          for (int f = 0; f < F; ++f) v[q][f] = ((const float4*)(from + 2 * S::ROWS + i * DP))[l16 + 16 * f];
        }
#pragma unroll
        for (int q = 0; q < U; ++q)
          if (p + q * step < n_parts) add(ml[q], v[q]);
      }
      if (many) {
        __syncthreads();  // the row before has been read
        if (l16 == 0) { s_ml[group][0] = m; s_ml[group][1] = l; }
#pragma unroll
        for (int f = 0; f < F; ++f) s_acc[group][l16 + 16 * f] = acc[f];
        __syncthreads();
        // The first wave ends the row, its first 16 lanes with what all groups have added up; the others stay for a row that is done again,
        // which takes a whole wave.
        if (wave) continue;
        if (group == 0) {
          for (int o = 1; o < PA_JOIN_GROUPS; ++o) {
            float4 v[F];
#pragma unroll
            for (int f = 0; f < F; ++f) v[f] = s_acc[o][l16 + 16 * f];
            add(make_float2(s_ml[o][0], s_ml[o][1]), v);
          }
        }
      }
      const bool holds = !many || group == 0;  // this lane has a row's sums
      const int r = note.tile * S::ROWS + i, tok = req.row0 + r / G, h = note.hk * G + r % G;
      bool fine = !holds || l == l;
      if (P.sinks && m != -INFINITY) l += exp2f(fmaf(P.sinks[h], 1.4426950408889634f, pa_weights<DT>::SCALE) - m);
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int d = 4 * l16 + 64 * f;
        if (!holds || d >= P.D) continue;
        const float4 o = make_float4(acc[f].x * inv, acc[f].y * inv, acc[f].z * inv, acc[f].w * inv);
        fine = fine && pa_fine<DT>(o.x) && pa_fine<DT>(o.y) && pa_fine<DT>(o.z) && pa_fine<DT>(o.w);
        char* to = (char*)P.out + ((int64_t)tok * P.os_t + (int64_t)h * P.os_h + d) * S::ES;
        if (DT == SAH_F32) *(float4*)to = o;
        else *(uint2*)to = make_uint2(sah_pack2_hw<DT>(o.x, o.y), sah_pack2_hw<DT>(o.z, o.w));
      }
      // rows that are not finite are done again, one after the other, by the wave that has them
      uint64_t again = __ballot(!fine);
      while (again) {
        const int from = __builtin_ctzll(again) & ~15;
        again &= ~(0xffffull << from);
        pa_row_again<DT>(P, req, note.b, __builtin_amdgcn_readlane(tok, from), __builtin_amdgcn_readlane(h, from));
      }
    }
  }
  if (!note.again) return;  // uniform
  // rows of whole tiles that came out not finite: the first kernel's walk once more
  const pa_piece piece = pa_start<PA_JOIN_NT, S>(P, w, s_sum);
  const int64_t x0 = piece.x0, x1 = piece.x1;
  pa_place at = piece.at;
  for (;;) {
    if (at.begin >= x0 && (at.begin + at.cost <= x1 || at.cost <= piece.whole)) {
      const int n_rows = at.req.n_new * G;
      for (int i = (int)blockIdx.y * NW + wave; i < S::ROWS; i += PA_JOIN_WGS * NW) {
        const int r = at.tile * S::ROWS + i;
        if (r >= n_rows) break;
        const int tok = at.req.row0 + r / G, h = at.hk * G + r % G;
        bool fine = true;
        for (int d = lane; d < P.D; d += SAH_WAVE)
          fine = fine && pa_fine<DT>(sah_load<DT>(P.out, (int64_t)tok * P.os_t + (int64_t)h * P.os_h + d));
        if (__ballot(!fine)) pa_row_again<DT>(P, at.req, at.b, tok, h);
      }
    }
    if (at.begin + at.cost >= x1) break;
    if (!pa_next<S>(P, at)) break;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// Tiles of 128 rows whose waves share the keys, or of 32 rows whose waves each take keys of their own: by the rows per request, on average.
// Up to 32 nothing is shared. Up to 64 half of a wide tile is empty, but a narrow one's end, where 8 waves are added up, counts where there are
// several a workgroup; up to 128 a wide tile costs nothing more, but has four times as much to join where few tiles are shared by all. In us,
// narrow / wide, 8 key heads of 128, bf16: 1 request of 64 rows and 32768 keys 41 / 59, 16 of 64 and 4096 50 / 52, 64 of 64 and 1024 66 / 46;
// 1 of 128 and 32768 52 / 64, 4 of 128 and 8192 49 / 47, 16 of 128 and 4096 83 / 65; 1 of 256 and 32768 79 / 69, of 8192 and 8192 434 / 260.
// fp32 is bound by its matrix instructions (a sixteenth of the 16-bit rate) however often keys are read: 32 rows, so that a
// request of few rows keeps all waves busy (5 requests of 4 to 132 rows, 2000 keys on average: 66 us as tiles of 128, 34 so).
static bool pa_wide(const sah_paged_attention_args* a) {
  const int64_t rows = (int64_t)a->n_tokens * (a->Hq / a->Hkv), n = a->n_requests, tiles = rows * a->Hkv / 32;
  if (a->dtype == SAH_F32 || rows <= 32 * n) return false;
  return tiles > (rows <= 64 * n ? 2 * PA_CUS : rows <= 128 * n ? PA_CUS / 4 : 0);
}

// About as many workgroups as the call has work for, at most what the card holds at once: a short call's idle ones, and theirs of the
// second kernel, cost it 0.3 to 0.6 us of 17. Only how the work is shared depends on it.
template <typename S>
static int pa_workgroups(const sah_paged_attention_args* a) {
  const int G = a->Hq / a->Hkv;
  const int64_t table = (int64_t)a->table_width * a->page_size;
  int64_t keys = a->max_context > 0 && a->max_context < table ? a->max_context : table;
  if (a->window && (int64_t)a->sink + a->window + S::ROWS < keys) keys = (int64_t)a->sink + a->window + S::ROWS;
  const double tiles = ((double)a->n_tokens * G / S::ROWS + a->n_requests) * a->Hkv;
  const double n = tiles * (double)(keys + S::TILE_COST) / S::LEAST;
  return n < S::WGS ? ((int)n / PA_XCDS + 1) * PA_XCDS : S::WGS;
}

// notes for all workgroups that fit the card, two parts for each that is launched
template <int DT, int DP, bool WIDE>
static int64_t pa_floats(const sah_paged_attention_args* a) {
  typedef pa_shape<DT, DP, WIDE> S;
  return S::WGS * (int64_t)(sizeof(pa_note) / 4) + 2 * (int64_t)pa_workgroups<S>(a) * S::SLOT;
}

template <int DT, int DP, bool WIDE>
static int pa_launch(const sah_paged_attention_args* a) {
  typedef pa_shape<DT, DP, WIDE> S;
  static_assert(S::WGS % PA_XCDS == 0, "workgroups are dealt to the XCDs in turn");
  const int wgs = pa_workgroups<S>(a);
  hipStream_t st = (hipStream_t)a->stream;
  {
    sah_timed timed("k_paged_attn", a->stream);
    hipLaunchKernelGGL((k_paged_attn<DT, DP, WIDE>), dim3(wgs), dim3(S::NT), 0, st, *a);
    if (int rc = sah_launch_status("sah_paged_attention")) return rc;
  }
  sah_timed timed("k_paged_attn_join", a->stream);
  hipLaunchKernelGGL((k_paged_attn_join<DT, DP, WIDE>), dim3(wgs, PA_JOIN_WGS), dim3(PA_JOIN_NT), 0, st, *a);
  return sah_launch_status("sah_paged_attention(join)");
}

// calls f with the instance that a call takes
template <typename F>
static int64_t pa_dispatch(const sah_paged_attention_args* a, F f) {
  const bool wide = pa_wide(a);
  const int dp = a->D <= 64 ? 64 : a->D <= 128 ? 128 : 256;
#define PA_CASE(dt, d) if (a->dtype == dt && dp == d) return wide ? f.template operator()<dt, d, true>() : f.template operator()<dt, d, false>();
  PA_CASE(SAH_BF16, 64) PA_CASE(SAH_BF16, 128) PA_CASE(SAH_BF16, 256)
  PA_CASE(SAH_F16, 64) PA_CASE(SAH_F16, 128) PA_CASE(SAH_F16, 256)
#undef PA_CASE
  if (dp == 64) return f.template operator()<SAH_F32, 64, false>();
  if (dp == 128) return f.template operator()<SAH_F32, 128, false>();
  return f.template operator()<SAH_F32, 256, false>();
}
struct pa_floats_fn {
  const sah_paged_attention_args* a;
  template <int DT, int DP, bool WIDE> int64_t operator()() const { return pa_floats<DT, DP, WIDE>(a); }
};
struct pa_launch_fn {
  const sah_paged_attention_args* a;
  template <int DT, int DP, bool WIDE> int64_t operator()() const { return pa_launch<DT, DP, WIDE>(a); }
};

extern "C" int64_t sah_paged_attention_work_floats(const sah_paged_attention_args* a) {
  if (!a || a->n_tokens <= 0 || a->n_requests <= 0 || a->Hkv <= 0 || a->Hq < a->Hkv || a->D <= 0 || a->D > PA_MAX_D || a->table_width <= 0 ||
      a->page_size <= 0)
    return 0;
  return pa_dispatch(a, pa_floats_fn{a});
}

extern "C" int sah_paged_attention(const sah_paged_attention_args* given) {
  if (!given) return sah_fail(SAH_ENULL, "sah_paged_attention: args is NULL");
  sah_paged_attention_args own = *given;
  const sah_paged_attention_args* a = &own;
  // a dimension of one entry has no stride, whatever it is said to be
  if (own.n_tokens == 1) own.qs_t = own.os_t = 0;
  if (own.Hq == 1) own.qs_h = own.os_h = 0;
  if (own.Hkv == 1) own.ks_h = own.vs_h = 0;
  if (own.n_pages == 1) own.ks_p = own.vs_p = 0;
  if (own.page_size == 1) own.ks_t = own.vs_t = own.D;
  if (a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16) return sah_fail(SAH_EDTYPE, "sah_paged_attention: dtype %d", a->dtype);
  if (a->n_requests <= 0 || a->n_tokens < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->n_pages <= 0 || a->table_width <= 0 ||
      a->max_context < 0 || a->sink < 0 || a->window < 0)
    return sah_fail(SAH_EINVAL, "sah_paged_attention: bad sizes (n_requests %d, n_tokens %d, heads %d / %d, n_pages %d, table_width %d, max_context %d, "
                    "sink %d, window %d)", a->n_requests, a->n_tokens, a->Hq, a->Hkv, a->n_pages, a->table_width, a->max_context, a->sink, a->window);
  if (a->D <= 0 || a->D % 8 || a->D > PA_MAX_D) return sah_fail(SAH_ESHAPE, "sah_paged_attention: head_dim %d is not a multiple of 8 up to 256", a->D);
  if (a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return sah_fail(SAH_ESHAPE, "sah_paged_attention: page_size %d is not a power of two", a->page_size);
  if ((int64_t)a->table_width * a->page_size > INT32_MAX - 4096)  // (a stage's keys reach beyond the last one)
    return sah_fail(SAH_ESHAPE, "sah_paged_attention: table_width * page_size passes 2^31 - 4097");
  if ((int64_t)a->n_tokens * a->Hq > 1 << 30) return sah_fail(SAH_ESHAPE, "sah_paged_attention: n_tokens * Hq passes 2^30");
  // the line of work is divided in doubles, also where running sums overlap
  if (((double)a->n_tokens * (a->Hq / a->Hkv) / 32 + 1) * ((double)a->table_width * a->page_size + 1024) * a->Hkv * a->n_requests > 0x1p52)
    return sah_fail(SAH_ESHAPE, "sah_paged_attention: too much work for one call");
  if (a->table_pitch < a->table_width) return sah_fail(SAH_EINVAL, "sah_paged_attention: table_pitch is less than table_width");
  if (a->n_tokens == 0) return SAH_OK;
  if (!a->q || !a->k || !a->v || !a->block_table || !a->kv_lens || !a->cu_new || !a->out) return sah_fail(SAH_ENULL, "sah_paged_attention: NULL pointer");
  const int es = a->dtype == SAH_F32 ? 4 : 2;
  if (((uint64_t)a->q | (uint64_t)a->k | (uint64_t)a->v | (uint64_t)a->out | (uint64_t)a->work |
       (uint64_t)(es * (a->qs_t | a->qs_h | a->ks_p | a->ks_t | a->ks_h | a->vs_p | a->vs_t | a->vs_h | a->os_t | a->os_h))) % 16)
    return sah_fail(SAH_EINVAL, "sah_paged_attention: addresses and strides must be multiples of 16 bytes");
  if (a->ks_t < 0 || a->vs_t < 0 || a->ks_t >= 1 << 26 || a->vs_t >= 1 << 26)  // a few tokens of a page: 32-bit offsets
    return sah_fail(SAH_ESHAPE, "sah_paged_attention: a page's tokens are 2^26 elements or more apart");
  if (!sah_rows_apart<2>(a->D, {a->os_t, a->os_h}, {a->n_tokens, a->Hq})) return sah_fail(SAH_EINVAL, "sah_paged_attention: rows of out overlap");
  if (!(a->scaling - a->scaling == 0.f)) return sah_fail(SAH_EINVAL, "sah_paged_attention: scaling is not finite");
  if (!a->work || a->work_floats < sah_paged_attention_work_floats(a)) return sah_fail(SAH_ECAPACITY, "sah_paged_attention: work is too small");
  // rows are read again after others have been written
  const sah_span out = sah_span_of<2>(a->out, es, a->D, {a->os_t, a->os_h}, {a->n_tokens, a->Hq});
  if (sah_out_on_queries(a->q, a->qs_t, a->qs_h, a->out, a->os_t, a->os_h, a->n_tokens, a->Hq, a->D, es)) return sah_fail(SAH_EINVAL, "sah_paged_attention: out shares memory with q");
  if (sah_meet(out, sah_span_of<3>(a->k, es, a->D, {a->ks_p, a->ks_t, a->ks_h}, {a->n_pages, a->page_size, a->Hkv})) ||
      sah_meet(out, sah_span_of<3>(a->v, es, a->D, {a->vs_p, a->vs_t, a->vs_h}, {a->n_pages, a->page_size, a->Hkv})) ||
      sah_meet(out, sah_span_of<1>(a->block_table, 4, a->table_width, {a->table_pitch}, {a->n_requests})) ||
      sah_meet(out, sah_span_of<1>(a->kv_lens, 4, 1, {1}, {a->n_requests})) || sah_meet(out, sah_span_of<1>(a->cu_new, 4, 1, {1}, {a->n_requests + 1})) ||
      (a->sinks && sah_meet(out, sah_span_of<1>(a->sinks, 4, 1, {1}, {a->Hq}))))
    return sah_fail(SAH_EINVAL, "sah_paged_attention: out lies within the cache, the table or the lengths");
  return (int)pa_dispatch(a, pa_launch_fn{a});
}
