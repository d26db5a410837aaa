// Attention over pages in 8 bits, or over the pages that a list names for each token: few rows a request, so that memory bounds it.
//
// Of a request's tokens (with a list: of one token) and a key head's query heads every (token, head) is a row; up to 16 are a tile.
// A workgroup has a tile and a stretch of the keys that it sees, its four waves take 32 keys of it in turn. Nothing is staged: keys and values
// go from memory to the registers in which the matrix instructions want them. S^T = K Q^T (16 keys x 16 rows a tile of the matrix): a lane reads 16
// bytes of a key's row, the 4 lanes of a key 64 neighbouring ones. The result has row n in lanes n + 16 g, keys 4 g .. 4 g + 3 of both key
// tiles, which is what O^T = V^T P^T wants of P with its key slots in that order; of V lane i + 16 g then holds the 8 keys' dims
// C i .. C i + C - 1 (a key's row is 16 lanes' pieces, one after the other), and a permutation of 16-bit halves inside the lane makes of
// them the operand of dim C i + e, the output's tile e. 8-bit elements become bf16 on the way, their scale with them, in one instruction a pair: exact.
// A 32-key step's K is requested as soon as the step before has been multiplied with its own, V likewise: half a step or more is under way at all times.
// Parts of a tile (m, l, acc) are joined by a second kernel.
#include "sah_pages.h"
#include "sah_spans.h"

#define PT_NT 256
#define PT_NW (PT_NT / SAH_WAVE)
#define PT_ROWS 16
#define PT_STEP 32                      // keys of a wave's step
#define PT_ROUND (PT_STEP * PT_NW)      // of a workgroup's
#define PT_MOST 2048                    // keys whose pages a workgroup looks up at once
#define PT_SPLITS 256                   // workgroups that share a tile, at most

struct pt_args {
  sah_page_attention_args a;
  int splits, stretch;    // workgroups that share a tile; keys of each, at least
  int tokens, blocks;     // tokens of a tile; tiles that a token's query heads of a key head make
  int unit;               // window: keys that begin and end with one
  int64_t groups;         // (token, block, split)
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

// Keys of a workgroup: more than planned where a request is longer than the caller said.
__device__ __forceinline__ int pt_stretch(const pt_args& A, int n) {
  const int each = (int)(((int64_t)n + A.splits - 1) / A.splits);
  return each <= A.stretch ? A.stretch : (int)(((int64_t)each + PT_ROUND - 1) / PT_ROUND * PT_ROUND);
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

// SMALL: pages of less than 16 tokens, where a 16-key tile's keys do not lie in one page
template <int KT, int QT, int DP, bool SMALL>
__global__ __launch_bounds__(PT_NT) void k_page_attn(pt_args A) {
  sah_touch_kernargs<sizeof(pt_args)>();
  const sah_page_attention_args& P = A.a;
  const sah_page_cache& C = P.cache;
  typedef pt_types<KT, QT> T;
  constexpr int ES = pg_size(KT), MT = T::MT;
  constexpr int KL = DP * ES / 64;                                    // 16-byte loads of a lane and key tile
  constexpr int NC = KT == SAH_E4M3 ? DP / 16 : KT == SAH_F32 ? 4 : DP >= 128 ? 8 : 4;  // elements of a lane's piece of a value row
  constexpr int H = DP / (16 * NC);                                   // pieces
  constexpr int VW = NC * ES / 4;                                     // 32-bit words of a piece
  constexpr int TILES = DP / 16;
  constexpr int PITCH = DP + 4;                                       // floats of a row in LDS
  constexpr int SLOTS = SMALL ? PT_MOST + PT_ROUND : PT_MOST / 16 + PT_ROUND / 16 + 2;
  __shared__ int s_page[SLOTS], s_first[SLOTS];                       // of the stretch's pages: number, first key
  __shared__ __align__(16) float s_acc[PT_NW][PT_ROWS][PITCH];
  __shared__ float s_ml[PT_NW][2][PT_ROWS];
  __shared__ uint32_t s_bad;

  // The key heads of a tile and stretch, whose tokens lie side by side, are on one XCD.
  const int64_t x = (int64_t)blockIdx.x / 8;
  const int64_t group = x / C.Hkv * 8 + blockIdx.x % 8;
  const int hk = (int)(x % C.Hkv);
  if (group >= A.groups) return;
  const int split = (int)(group % A.splits);
  const int64_t tb = group / A.splits;
  const int block = (int)(tb % A.blocks), t0 = (int)(tb / A.blocks);
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id(), i16 = lane & 15, g = lane >> 4;
  const pg_request req = pg_find_by_wave(P.requests, C.page_size, t0);
  if (req.b < 0) return;
  const int G = P.Hq / C.Hkv, i0 = t0 - req.begin;
  if (A.tokens > 1 && i0 % A.tokens) return;   // not the first of its tile
  const int n_tok = A.tokens < req.n_new - i0 ? A.tokens : req.n_new - i0;
  const int rows = A.blocks > 1 ? (G - block * PT_ROWS < PT_ROWS ? G - block * PT_ROWS : PT_ROWS) : n_tok * G;
  const int64_t p_lo = req.base + t0, p_hi = p_lo + n_tok - 1;
  const pt_keys keys = pt_keys_of(A, req, p_lo, p_hi);
  const int stretch = pt_stretch(A, keys.n);
  const int64_t begin = (int64_t)split * stretch;
  if (A.splits > 1 && begin >= keys.n) return;  // (the joining knows)
  const int u_first = (int)begin, u_end = keys.n - u_first < stretch ? keys.n : u_first + stretch;
  const int shift = 31 - __builtin_clz(C.page_size);
  const bool live = i16 < rows;
  const int rr = live ? i16 : rows - 1;
  const int tok = t0 + (A.blocks > 1 ? 0 : rr / G), head = hk * G + (A.blocks > 1 ? block * PT_ROWS + rr : rr % G);
  const int64_t p = req.base + tok;
  const int last = p < keys.hi ? (p < -1 ? -1 : (int)p) : keys.hi;          // the last key that this lane's row sees
  const int least = p_lo < keys.hi ? (p_lo < -1 ? -1 : (int)p_lo) : keys.hi; // ... that all rows see

  if (threadIdx.x == 0) s_bad = 0;
  // queries as the second operand, in the order in which a lane's 16 bytes of a key come
  const char* qp = (const char*)P.q + ((int64_t)tok * P.qs_t + (int64_t)head * P.qs_h) * pg_size(QT);
  const float sign = P.scaling < 0.f ? -1.f : 1.f;
  uint4 qf[T::NQ][KT == SAH_F32 ? KL : DP / 32];
#pragma unroll
  for (int s = 0; s < (KT == SAH_F32 ? KL : DP / 32); ++s) {
    constexpr int E = KT == SAH_F32 ? 4 : 8;
    const int d = KT == SAH_F32 ? 16 * s + 4 * g : KT == SAH_E4M3 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (d < C.D && live) {
      if constexpr (KT == SAH_F32) {
        const float4 f = *(const float4*)(qp + 4 * d);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
      } else {
        sah_load8<QT>(qp, d, v);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= sign;
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

  const float c_exp = pt_log2(P.scaling);
  float m_run = -INFINITY, l_run = 0.f;
  sah_f32x4 acc[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;

  // what lies behind a shorter head's end is its last piece again: the queries are 0 there, the results nobody's
  int k_in[KL];
#pragma unroll
  for (int s = 0; s < KL; ++s) {
    const int at = 64 * s + 16 * g;
    k_in[s] = at < C.D * ES ? at : C.D * ES - 16;
  }
  int v_in[H];
#pragma unroll
  for (int s = 0; s < H; ++s) {
    const int at = (s * 16 + i16) * NC;
    v_in[s] = (at < C.D ? at : C.D - NC) * ES;
  }
  const char* kbase = (const char*)C.k + (int64_t)hk * C.ks_h * ES;
  const char* vbase = (const char*)C.v + (int64_t)hk * C.vs_h * ES;
  const int kt = (int)(C.ks_t * ES), vt = (int)(C.vs_t * ES);   // (less than 2^28)

  sah_u4 kr[2][KL];
  uint32_t vr[H][8][VW];
  uint32_t k_scale[2], v_scale[2];   // bytes: of this lane's key in a tile; of its four
  int u0 = u_first;  // of what s_page and s_first hold
  auto slot_of = [&](int u) { return (u - u0 + (u0 & (C.page_size - 1))) >> shift; };
  auto in_page = [&](int u) { return u & (C.page_size - 1); };
  auto fetch_k = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const char* at;
      if constexpr (SMALL) {
        const int key = u + 16 * a + i16, page = s_page[slot_of(key)], in = in_page(key);
        at = kbase + (page * C.ks_p + in * C.ks_t) * ES;
        if constexpr (KT == SAH_E4M3) k_scale[a] = C.k_scales[((int64_t)page * C.Hkv + hk) * C.page_size + in];
      } else {
        const int64_t page = __builtin_amdgcn_readfirstlane(s_page[slot_of(u + 16 * a)]);
        const int in = in_page(u + 16 * a);
        at = kbase + (page * C.ks_p + in * C.ks_t) * ES + (int64_t)i16 * kt;
        if constexpr (KT == SAH_E4M3) k_scale[a] = C.k_scales[(page * C.Hkv + hk) * C.page_size + in + i16];
      }
#pragma unroll
      for (int s = 0; s < KL; ++s) kr[a][s] = *(const sah_u4*)(at + k_in[s]);
    }
  };
  auto fetch_v = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const char* at = nullptr;
      if constexpr (!SMALL) {
        const int64_t page = __builtin_amdgcn_readfirstlane(s_page[slot_of(u + 16 * a)]);
        const int in = in_page(u + 16 * a);
        at = vbase + (page * C.vs_p + in * C.vs_t) * ES + (int64_t)(4 * g) * vt;
        if constexpr (KT == SAH_E4M3) v_scale[a] = *(const uint32_t*)(C.v_scales + (page * C.Hkv + hk) * C.page_size + in + 4 * g);
      } else if constexpr (KT == SAH_E4M3) {
        v_scale[a] = 0;
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const char* row;
        if constexpr (SMALL) {
          const int key = u + 16 * a + 4 * g + v, page = s_page[slot_of(key)], in = in_page(key);
          row = vbase + (page * C.vs_p + in * C.vs_t) * ES;
          if constexpr (KT == SAH_E4M3) v_scale[a] |= (uint32_t)C.v_scales[((int64_t)page * C.Hkv + hk) * C.page_size + in] << (8 * v);
        } else {
          row = at + (int64_t)v * vt;
        }
#pragma unroll
        for (int s = 0; s < H; ++s) {
          const char* from = row + v_in[s];
          uint32_t* to = vr[s][4 * a + v];
          if constexpr (VW == 4) {
            const sah_u4 w = *(const sah_u4*)from;
            to[0] = w.x; to[1] = w.y; to[2] = w.z; to[3] = w.w;
          } else if constexpr (VW == 2) {
            const sah_u2 w = *(const sah_u2*)from;
            to[0] = w.x; to[1] = w.y;
          } else {
            to[0] = *(const uint32_t*)from;
          }
        }
      }
    }
  };

  auto step = [&](int u, auto k_read, auto v_read) __attribute__((always_inline)) {
    sah_f32x4 s[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[a][e] = 0.f;
      const float scale = KT == SAH_E4M3 ? pg_scale(k_scale[a]) : 1.f;
#pragma unroll
      for (int c = 0; c < KL; ++c) {
        const sah_u4 k = kr[a][c];
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
    k_read();
    // keys that not every row sees; values of keys that no row sees are made 0
    bool plain = true;   // uniform
    if constexpr (!SMALL) {
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int first = __builtin_amdgcn_readfirstlane(s_first[slot_of(u + 16 * a)]) + in_page(u + 16 * a);
        plain = plain && first + 15 <= least && (!P.window || first + 15 < P.sink || first > p_hi - P.window);
      }
    } else {
      plain = false;
    }
    if (!plain) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = u + 16 * a + 4 * g + e;
          const int j = s_first[slot_of(key)] + in_page(key);
          const bool on = j <= last && (!P.window || j < P.sink || j > p - P.window);
          const bool some = j <= keys.hi && (!P.window || j < P.sink || j > p_lo - P.window);
          s[a][e] = on ? s[a][e] : -INFINITY;
#pragma unroll
          for (int c = 0; c < H; ++c)
#pragma unroll
            for (int w = 0; w < VW; ++w) vr[c][4 * a + e][w] = some ? vr[c][4 * a + e][w] : 0u;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int a = 0; a < 2; ++a)
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
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[a][e] = __builtin_amdgcn_exp2f(fmaf(s[a][e] - m_at, c_exp, T::SCALE));
        l_run += s[a][e];
      }
    if constexpr (KT == SAH_F32) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int c = 0; c < H; ++c)
#pragma unroll
            for (int w = 0; w < NC; ++w) acc[c * NC + w] = pt_mfma_f32(sah_bits_to_float(vr[c][4 * a + e][w]), s[a][e], acc[c * NC + w]);
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
              const float scale = pg_scale_of(v_scale[k / 4], k % 4);
              two[k] = pair % 2 ? pg_widen2<true>(vr[c][k][pair / 2], scale) : pg_widen2<false>(vr[c][k][pair / 2], scale);
            } else {
              two[k] = vr[c][k][pair];
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
    v_read();
  };
  for (; u0 < u_end; u0 += PT_MOST) {  // (uniform; the next one's first key fits 32 bits: the host has checked what a request can have)
    const int u1 = u_end - u0 < PT_MOST ? u_end : u0 + PT_MOST;
    if (u0 != u_first) __syncthreads();   // the pages before have been read
    const int n_slots = ((u1 - u0 + PT_STEP - 1) / PT_STEP * PT_STEP - 1 + (u0 & (C.page_size - 1))) >> shift;
    const int32_t* list = P.pages ? P.pages + ((int64_t)t0 * C.Hkv + hk) * P.n_select : nullptr;
    for (int s = threadIdx.x; s <= n_slots; s += PT_NT) {
      const int e = (u0 >> shift) + s;
      int lg = e;
      if (list) lg = e < P.n_select ? list[e] : -1;
      else if (keys.skip && e >= keys.sinks >> shift) lg = e + (keys.skip >> shift);
      int page = -1;
      if (lg >= 0 && lg < P.requests.table_width && lg <= keys.hi >> shift) page = P.requests.block_table[(int64_t)req.b * P.requests.table_pitch + lg];
      const bool there = page >= 0 && page < C.n_pages;
      s_page[s] = there ? page : 0;
      s_first[s] = there ? lg << shift : (int)(0x80000000u - (uint32_t)C.page_size);  // (behind every position: table_width pages end before it)
    }
    __syncthreads();
    int u = u0 + PT_STEP * wave;
    if (u >= u1) continue;
    fetch_k(u);
    fetch_v(u);
    // (the last step apart: a way through the loop that skips a request would have the compiler wait for all of them)
#pragma unroll 1
    for (; u + PT_ROUND < u1; u += PT_ROUND)
      step(u, [&]() __attribute__((always_inline)) { fetch_k(u + PT_ROUND); }, [&]() __attribute__((always_inline)) { fetch_v(u + PT_ROUND); });
    step(u, [] {}, [] {});
  }

  // the four waves' sums, row by row in LDS (s_bad is set behind the wait)
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
  for (int i = threadIdx.x; i < rows * (DP / 4); i += PT_NT) {
    const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < PT_NW; ++w) m = fmaxf(m, s_ml[w][0][r]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < PT_NW; ++w) {
      const float mw = s_ml[w][0][r], lw = s_ml[w][1][r], up = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - m) * c_exp);
      l += lw == lw ? lw * up : lw;  // (a wave whose sum is NaN has no maximum, perhaps)
      const float4 a = *(const float4*)&s_acc[w][r][d];
      o.x += a.x * up;
      o.y += a.y * up;
      o.z += a.z * up;
      o.w += a.w * up;
    }
    const int rt = t0 + (A.blocks > 1 ? 0 : r / G), rh = hk * G + (A.blocks > 1 ? block * PT_ROWS + r : r % G);
    if (A.splits > 1) {
      float* to = (float*)P.work + (((int64_t)rt * P.Hq + rh) * A.splits + split) * (DP + 4);
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
    if (!fine) atomicOr(&s_bad, 1u << r);
    char* to = (char*)P.out + ((int64_t)rt * P.os_t + (int64_t)rh * P.os_h + d) * pg_size(QT);
    if (QT == SAH_F32) *(float4*)to = o;
    else *(uint2*)to = make_uint2(sah_pack2_hw<QT>(o.x, o.y), sah_pack2_hw<QT>(o.z, o.w));
  }
  if (A.splits > 1) return;
  __syncthreads();
  uint32_t bad = s_bad;  // rows that are not finite are done again, each by a wave
  for (int i = 0; bad; ++i) {
    const int r = __builtin_ctz(bad);
    bad &= bad - 1;
    if (i % PT_NW != wave) continue;
    pt_row_again<KT, QT>(A, req, t0 + (A.blocks > 1 ? 0 : r / G), hk * G + (A.blocks > 1 ? block * PT_ROWS + r : r % G));
  }
}

// Joins the parts of the rows: a wave has a row, a lane DP / 64 of its dims.
#define PT_JOIN_U 8
template <int KT, int QT, int DP>
__global__ __launch_bounds__(PT_NT) void k_page_attn_join(pt_args A) {
  sah_touch_kernargs<sizeof(pt_args)>();
  const sah_page_attention_args& P = A.a;
  const sah_page_cache& C = P.cache;
  typedef pt_types<KT, QT> T;
  constexpr int F = DP / 64;
  const int lane = threadIdx.x & (SAH_WAVE - 1);
  const int64_t row = (int64_t)blockIdx.x * PT_NW + sah_wave_id();
  if (row >= (int64_t)P.requests.n_tokens * P.Hq) return;
  const int t = (int)(row / P.Hq), h = (int)(row - (int64_t)t * P.Hq);
  const pg_request req = pg_find_by_wave(P.requests, C.page_size, t);
  if (req.b < 0) return;
  const int i = t - req.begin, i0 = i - i % A.tokens, n_tok = A.tokens < req.n_new - i0 ? A.tokens : req.n_new - i0;
  const int64_t p_lo = req.base + req.begin + i0;
  const pt_keys keys = pt_keys_of(A, req, p_lo, p_lo + n_tok - 1);
  const int stretch = pt_stretch(A, keys.n), parts = (int)(((int64_t)keys.n + stretch - 1) / stretch);
  const float* from = (const float*)P.work + row * A.splits * (DP + 4);
  const float c_exp = pt_log2(P.scaling);
  float m = -INFINITY, l = 0.f, o[F];
#pragma unroll
  for (int f = 0; f < F; ++f) o[f] = 0.f;
  for (int p0 = 0; p0 < parts; p0 += PT_JOIN_U) {
    float2 ml[PT_JOIN_U];
    float v[PT_JOIN_U][F];
#pragma unroll
    for (int i = 0; i < PT_JOIN_U; ++i) {
      const float* part = from + (int64_t)(p0 + i < parts ? p0 + i : parts - 1) * (DP + 4);
      ml[i] = *(const float2*)part;
#pragma unroll
      for (int f = 0; f < F; ++f) v[i][f] = part[4 + lane * F + f];
    }
#pragma unroll
    for (int i = 0; i < PT_JOIN_U; ++i) {
      if (p0 + i >= parts) continue;
      const float m_new = fmaxf(m, ml[i].x);
      const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - m_new) * c_exp);
      const float z = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[i].x - m_new) * c_exp);
      l = l * a + (ml[i].y == ml[i].y ? ml[i].y * z : ml[i].y);
      m = m_new;
#pragma unroll
      for (int f = 0; f < F; ++f) o[f] = o[f] * a + v[i][f] * z;
    }
  }
  bool fine = l == l;
  if (P.sinks && m != -INFINITY) l += __builtin_amdgcn_exp2f(fmaf(P.sinks[h], 1.4426950408889634f, T::SCALE) - m * c_exp);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int d = lane * F + f;
    if (d >= C.D) continue;
    o[f] *= inv;
    fine = fine && pt_fine<QT>(o[f]);
    sah_store<QT>(P.out, (int64_t)t * P.os_t + (int64_t)h * P.os_h + d, o[f]);
  }
  if (__ballot(!fine)) pt_row_again<KT, QT>(A, req, t, h);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// How a call's tiles are shared. About PT_WGS workgroups, if that leaves each a round of keys; no more than PT_MOST keys of each, so that requests of uneven
// lengths keep the card busy, but where there are many tiles.
#define PT_WGS 1024
static pt_args pt_plan(const sah_page_attention_args* a) {
  pt_args A;
  A.a = *a;
  const int G = a->Hq / a->cache.Hkv;
  A.tokens = a->pages || G >= PT_ROWS ? 1 : PT_ROWS / G;
  A.blocks = (G + PT_ROWS - 1) / PT_ROWS;
  A.unit = a->cache.page_size > PT_STEP ? a->cache.page_size : PT_STEP;
  const int64_t table = (int64_t)a->requests.table_width * a->cache.page_size;
  int64_t most = table;   // keys that a tile may see
  if (a->pages) most = (int64_t)a->n_select * a->cache.page_size;
  else if (a->window) {
    const int64_t w = ((int64_t)a->sink + A.unit - 1) / A.unit * A.unit + a->window + A.tokens + 2 * (int64_t)A.unit;
    most = w < table ? w : table;
  }
  int64_t usual = most;   // ... about, by what the caller says
  if (!a->pages && a->max_context > 0 && a->max_context < usual) usual = a->max_context;
  const double tiles = ((double)a->requests.n_tokens / A.tokens + (A.tokens > 1 ? a->requests.n_requests : 0)) * A.blocks * a->cache.Hkv;
  const double limit = tiles > 4 * PT_WGS ? PT_MOST * tiles / (4 * PT_WGS) : PT_MOST;
  const double each = fmin(tiles * (double)usual / PT_WGS, limit);
  A.stretch = (int)((int64_t)(fmin(each, 1e9) + PT_ROUND - 1) / PT_ROUND * PT_ROUND);
  if (A.stretch < PT_ROUND) A.stretch = PT_ROUND;
  const int64_t splits = (usual + A.stretch - 1) / A.stretch;
  A.splits = (int)(splits < 1 ? 1 : splits < PT_SPLITS ? splits : PT_SPLITS);
  A.groups = (int64_t)a->requests.n_tokens * A.blocks * A.splits;
  return A;
}

// Chunks of an 8-bit cache: bytes of the copies of K and V and of their table, and the call on them; 0 where the cache is attended to as it is.
static int64_t pt_copy_bytes(const sah_page_attention_args* a) {
  if (a->pages || a->cache.dtype != SAH_E4M3) return 0;
  const int64_t rows = (int64_t)a->requests.n_tokens * (a->Hq / a->cache.Hkv);
  if (rows <= 32 * (int64_t)a->requests.n_requests) return 0;
  const double pages = (double)a->requests.n_requests * a->requests.table_width;
  const double bytes = pages * a->cache.page_size * a->cache.Hkv * a->cache.D * pg_size(a->dtype) * 2;
  if (bytes > 0x1p33 || pages * 4 > 0x1p33) return 0;
  return (int64_t)bytes + ((int64_t)pages * 4 + 15) / 16 * 16;
}
static sah_paged_attention_args pt_on_copy(const sah_page_attention_args* a) {
  const sah_page_cache& c = a->cache;
  sah_paged_attention_args p = {};
  const int64_t row = c.D, token = row * c.Hkv, page = token * c.page_size, pages = (int64_t)a->requests.n_requests * a->requests.table_width;
  const int es = pg_size(a->dtype);
  char* k = (char*)a->work;
  p.q = a->q; p.qs_t = a->qs_t; p.qs_h = a->qs_h;
  p.k = k; p.ks_p = page; p.ks_t = token; p.ks_h = row;
  p.v = k + pages * page * es; p.vs_p = page; p.vs_t = token; p.vs_h = row;
  p.block_table = (const int32_t*)(k + 2 * pages * page * es);
  p.table_pitch = p.table_width = a->requests.table_width;
  p.kv_lens = a->requests.kv_lens;
  p.cu_new = a->requests.cu_new;
  p.sinks = a->sinks;
  p.dtype = a->dtype;
  p.n_requests = a->requests.n_requests; p.n_tokens = a->requests.n_tokens; p.Hq = a->Hq; p.Hkv = c.Hkv; p.D = c.D;
  p.n_pages = (int)pages; p.page_size = c.page_size;
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
  if (const int64_t copy = pt_copy_bytes(a)) {
    const sah_paged_attention_args p = pt_on_copy(a);
    return copy + 4 * sah_paged_attention_work_floats(&p);
  }
  const pt_args A = pt_plan(a);
  return A.splits > 1 ? (int64_t)a->requests.n_tokens * a->Hq * A.splits * (pt_dim(a) + 4) * 4 : 0;
}

template <int KT, int QT, int DP>
static int pt_launch(const pt_args& A, unsigned wgs) {
  hipStream_t st = (hipStream_t)A.a.stream;
  {
    sah_timed timed("k_page_attn", A.a.stream);
    if (A.a.cache.page_size < 16) hipLaunchKernelGGL((k_page_attn<KT, QT, DP, true>), dim3(wgs), dim3(PT_NT), 0, st, A);
    else hipLaunchKernelGGL((k_page_attn<KT, QT, DP, false>), dim3(wgs), dim3(PT_NT), 0, st, A);
    if (int rc = sah_launch_status("sah_page_attention")) return rc;
  }
  if (A.splits == 1) return SAH_OK;
  sah_timed timed("k_page_attn_join", A.a.stream);
  const int64_t rows = (int64_t)A.a.requests.n_tokens * A.a.Hq;
  hipLaunchKernelGGL((k_page_attn_join<KT, QT, DP>), dim3((unsigned)((rows + PT_NW - 1) / PT_NW)), dim3(PT_NT), 0, st, A);
  return sah_launch_status("sah_page_attention(join)");
}
template <int KT, int QT>
static int pt_launch_dim(const pt_args& A, unsigned wgs) {
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
  if ((a->pages != nullptr) != (a->n_select > 0)) return sah_fail(SAH_EINVAL, "sah_page_attention: pages and n_select go together");
  if (a->pages && (a->window || a->sink)) return sah_fail(SAH_EINVAL, "sah_page_attention: pages and a window do not go together");
  if (!a->pages && c.dtype != SAH_E4M3) return sah_fail(SAH_EDTYPE, "sah_page_attention: neither pages nor an 8-bit cache: sah_paged_attention's");
  if (int rc = pg_check_requests(r, c.page_size, true, what)) return rc;
  if ((int64_t)a->n_select * c.page_size > INT32_MAX - 4096) return sah_fail(SAH_ESHAPE, "sah_page_attention: n_select * page_size passes 2^31 - 4097");
  if ((int64_t)r.n_tokens * a->Hq > 1 << 30) return sah_fail(SAH_ESHAPE, "sah_page_attention: n_tokens * Hq passes 2^30");
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
  const int ces = pg_size(c.dtype);
  const int64_t scales = c.dtype == SAH_E4M3 ? (int64_t)c.n_pages * c.Hkv * c.page_size : 0;
  if (sah_meet(out, sah_span_of<3>(c.k, ces, c.D, {c.ks_p, c.ks_t, c.ks_h}, {c.n_pages, c.page_size, c.Hkv})) ||
      sah_meet(out, sah_span_of<3>(c.v, ces, c.D, {c.vs_p, c.vs_t, c.vs_h}, {c.n_pages, c.page_size, c.Hkv})) ||
      (scales && (sah_meet(out, sah_span_of<1>(c.k_scales, 1, scales, {0}, {1})) || sah_meet(out, sah_span_of<1>(c.v_scales, 1, scales, {0}, {1})))) ||
      sah_meet(out, sah_span_of<1>(r.block_table, 4, r.table_width, {r.table_pitch}, {r.n_requests})) ||
      sah_meet(out, sah_span_of<1>(r.kv_lens, 4, 1, {1}, {r.n_requests})) || sah_meet(out, sah_span_of<1>(r.cu_new, 4, 1, {1}, {r.n_requests + 1})) ||
      (a->pages && sah_meet(out, sah_span_of<1>(a->pages, 4, (int64_t)r.n_tokens * c.Hkv * a->n_select, {0}, {1}))) ||
      (a->sinks && sah_meet(out, sah_span_of<1>(a->sinks, 4, 1, {1}, {a->Hq}))))
    return sah_fail(SAH_EINVAL, "sah_page_attention: out lies within the cache, the table, the lists or the lengths");
  if (const int64_t copy = pt_copy_bytes(a)) {
    sah_paged_attention_args p = pt_on_copy(a);
    const int64_t row = c.D, token = row * c.Hkv, request = token * c.page_size * r.table_width;
    if (int rc = pg_load(c, r, a->dtype, pg_load_out{(void*)p.k, (void*)p.v, request, row, token, r.table_width * c.page_size, (int32_t*)p.block_table},
                         a->stream, what))
      return rc;
    p.work = (float*)((char*)a->work + copy);
    p.work_floats = (a->work_bytes - copy) / 4;
    return sah_paged_attention(&p);
  }
  const pt_args A = pt_plan(a);
  const int64_t wgs = (A.groups + 7) / 8 * 8 * c.Hkv;
  if (wgs > 0x7fffffff) return sah_fail(SAH_ESHAPE, "sah_page_attention: too much work for one call");
  if (c.dtype == SAH_F32) return pt_launch_dim<SAH_F32, SAH_F32>(A, (unsigned)wgs);
  if (c.dtype == SAH_BF16) return pt_launch_dim<SAH_BF16, SAH_BF16>(A, (unsigned)wgs);
  if (c.dtype == SAH_F16) return pt_launch_dim<SAH_F16, SAH_F16>(A, (unsigned)wgs);
  if (a->dtype == SAH_F32) return pt_launch_dim<SAH_E4M3, SAH_F32>(A, (unsigned)wgs);
  if (a->dtype == SAH_BF16) return pt_launch_dim<SAH_E4M3, SAH_BF16>(A, (unsigned)wgs);
  return pt_launch_dim<SAH_E4M3, SAH_F16>(A, (unsigned)wgs);
}
