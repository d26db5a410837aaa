// A paged cache in 8 bits: tokens quantised into their slots, contexts read back. Bounds of pages, and the pages that a token attends to.
#include "sah_pages.h"

#define PG_NT 256
#define PG_LOAD_WGS 16384
#define PG_BOUND_WAVES 4096

// ---------------------------------------------------------------------------
// store: 16 lanes hold a row (token, key head) of both matrices, 8 elements each (16 beyond 128 dims)
// Memory bounds it: 16384 tokens of 8 heads of 128 in bf16, 101 MB, 24 us (a large copy's rate: 21). Keys and values by one thread, so that the slot is
// read once and twice as many loads are under way: by a thread each 30.1 us.
// ---------------------------------------------------------------------------
// exponent of the scale of a row whose largest magnitude is `most`: the least e >= -110 with most <= 448 * 2^e = 1.75 * 2^(e + 8)
__device__ __forceinline__ int pg_exponent(float most) {
  const uint32_t bits = sah_float_to_bits(most);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);  // (a subnormal's field is 0: far below -110)
  return e > -110 ? e : -110;
}
__device__ __forceinline__ float pg_row16_max(float v) {
  v = fmaxf(v, sah_dpp<0xB1>(v));
  v = fmaxf(v, sah_dpp<0x4E>(v));
  v = fmaxf(v, sah_dpp<0x141>(v));
  return fmaxf(v, sah_dpp<0x140>(v));
}
// (the converter rounds to the nearest, ties to even, and gives NaN for what is not finite)
__device__ __forceinline__ uint32_t pg_narrow4(float a, float b, float c, float d) {
#if defined(__HIP_DEVICE_COMPILE__)
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
#else
  return 0;
#endif
}

template <int T>
__global__ __launch_bounds__(PG_NT) void k_page_store(sah_page_store_args P) {
  sah_touch_kernargs<sizeof(sah_page_store_args)>();
  constexpr int ES = pg_size(T);
  const sah_page_cache& C = P.cache;
  const int64_t row = (int64_t)blockIdx.x * (PG_NT / 16) + threadIdx.x / 16;
  const int l16 = threadIdx.x & 15;
  const int64_t t = row / C.Hkv;
  const int h = (int)(row - t * C.Hkv);
  if (t >= P.n_tokens) return;  // (all 16 lanes of a row go the same way)
  const char* from[2] = {(const char*)P.k + (t * P.ks_t + h * P.ks_h) * ES, (const char*)P.v + (t * P.vs_t + h * P.vs_h) * ES};
  float x[2][2][8];  // keys and values, requested with the slot
#pragma unroll
  for (int v = 0; v < 2; ++v)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = 8 * l16 + 128 * i;
      if (d < C.D) {
        sah_load8<T>(from[v], d, x[v][i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[v][i][e] = 0.f;
      }
    }
  const int64_t slot = P.slot_map[t];
  if (slot < 0 || slot >= (int64_t)C.n_pages * C.page_size) return;
  const int shift = 31 - __builtin_clz(C.page_size);
  const int64_t page = slot >> shift, entry = slot & (C.page_size - 1), scale = (page * C.Hkv + h) * C.page_size + entry;
  uint8_t* to[2] = {(uint8_t*)C.k + page * C.ks_p + entry * C.ks_t + h * C.ks_h, (uint8_t*)C.v + page * C.vs_p + entry * C.vs_t + h * C.vs_h};
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = fabsf(x[v][i][e]);
        most = fmaxf(most, a < INFINITY ? a : 0.f);
      }
    const int e = pg_exponent(pg_row16_max(most));
    const float up = sah_bits_to_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = 8 * l16 + 128 * i;
      if (d >= C.D) continue;
      const float* y = x[v][i];
      *(uint2*)(to[v] + d) = make_uint2(pg_narrow4(y[0] * up, y[1] * up, y[2] * up, y[3] * up), pg_narrow4(y[4] * up, y[5] * up, y[6] * up, y[7] * up));
    }
    if (l16 == 0) (v ? C.v_scales : C.k_scales)[scale] = (uint8_t)(e + 127);
  }
}

// ---------------------------------------------------------------------------
// load: a thread holds 8 elements of the cache (8-bit: what 16 bytes of a 16-bit result take) or 16 bytes of it (others: copied as they are)
// Memory bounds it: 24575 tokens of 8 heads of 128 in four contexts of up to 8192, 50 MB, to bf16, 134 MB with the zeros: 29 us, 6.5 TB/s. (Written
// through the L2: 33.8, with 16 elements a thread 36.4.)
// ---------------------------------------------------------------------------
// 16 bytes of a result: past the L2 where it is the caller's (ONCE), of which it would hold a small part and displace what the next kernel reads (24575 tokens
// read back 29 us, through it 35; the store after it 24, 28), through it where the attention reads it next.
template <bool ONCE>
__device__ __forceinline__ void pg_put16(char* to, sah_u4 x) {
  if constexpr (ONCE) __builtin_nontemporal_store(x, (sah_u4*)to);
  else *(sah_u4*)to = x;
}
// what 8 elements of e4m3 are in type T, stored at `to`
template <int T, bool ONCE>
__device__ __forceinline__ void pg_put8(char* to, uint2 x, float scale) {
  if constexpr (T == SAH_BF16) {
    pg_put16<ONCE>(to, sah_u4{pg_widen2<false>(x.x, scale), pg_widen2<true>(x.x, scale), pg_widen2<false>(x.y, scale), pg_widen2<true>(x.y, scale)});
  } else {
    float f[2][4];
    pg_widen4(x.x, scale, f[0]);
    pg_widen4(x.y, scale, f[1]);
    if constexpr (T == SAH_F32) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pg_put16<ONCE>(to + 16 * i, sah_u4{sah_float_to_bits(f[i][0]), sah_float_to_bits(f[i][1]), sah_float_to_bits(f[i][2]), sah_float_to_bits(f[i][3])});
    } else {
      // (a row's largest may have been rounded up past the type's; NaN stays)
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i / 4][i % 4] = f[i / 4][i % 4] > 65504.f ? 65504.f : (f[i / 4][i % 4] < -65504.f ? -65504.f : f[i / 4][i % 4]);
      pg_put16<ONCE>(to, sah_u4{sah_pack2_hw<SAH_F16>(f[0][0], f[0][1]), sah_pack2_hw<SAH_F16>(f[0][2], f[0][3]), sah_pack2_hw<SAH_F16>(f[1][0], f[1][1]),
                                sah_pack2_hw<SAH_F16>(f[1][2], f[1][3])});
    }
  }
}
// Whether one of 8 elements of e4m3 is a number that fp16 does not hold. All of them are multiples of 2^(e - 9) up to 448 * 2^e: from e = -15 to 7 none is.
__device__ __forceinline__ bool pg_none_of_f16(uint2 x, uint32_t scale) {
  if (scale >= 127 - 15 && scale <= 127 + 7) return false;
  float f[2][4];
  pg_widen4(x.x, pg_scale(scale), f[0]);
  pg_widen4(x.y, pg_scale(scale), f[1]);
  bool lost = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = f[i / 4][i % 4];
    lost |= v == v && (fabsf(v) > 65504.f || sah_f16_to_float(sah_float_to_f16(v)) != v);
  }
  return lost;
}
// CT: type of the cache; OT: of the output (other caches than SAH_E4M3: the same). `wgs` workgroups a request, which go through its tokens in
// turn: what lies behind a context in a table of a hundred thousand tokens costs a copy nothing. COPY: for the attention, with a table; requests without a row
// have no use for one (a chunk of 1024 tokens over 4024 keys beside 7 contexts of 32768 without one: 109 us, with copies of theirs 377).
template <int CT, int OT, bool COPY>
__global__ __launch_bounds__(PG_NT) void k_page_load(sah_page_cache C, sah_page_requests R, pg_load_out O, int wgs) {
  sah_touch_kernargs<sizeof(sah_page_cache) + sizeof(sah_page_requests) + sizeof(pg_load_out) + 4>();
  constexpr int CS = pg_size(CT), OS = pg_size(OT), E = CT == SAH_E4M3 ? 8 : 16 / CS;  // elements of a unit
  const uint32_t units = C.D / E, unit_h = units * C.Hkv, stride = (uint32_t)wgs * PG_NT, stride_t = stride / unit_h, stride_in = stride - stride_t * unit_h;
  const int shift = 31 - __builtin_clz(C.page_size), b = (int)blockIdx.x / wgs, kv = R.kv_lens[b];
  const int copied = O.length >> shift;  // pages of a copy
  if constexpr (COPY) {
    const int begin = R.cu_new[b], end = R.cu_new[b + 1];
    const bool idle = (begin > 0 ? begin : 0) >= (end < R.n_tokens ? end : R.n_tokens);
    if (idle || (O.first && O.first[b] < 0)) {
      if (O.lost && threadIdx.x == 0) O.lost[blockIdx.x] = !idle;
      return;
    }
  }
  const int64_t page0 = COPY && O.first ? O.first[b] : (int64_t)b * copied;
  [[maybe_unused]] bool lost = kv > O.length && R.table_width > copied;
  const uint32_t n = COPY && kv < O.length ? (kv > 0 ? kv : 0) : O.length, first = (blockIdx.x - (uint32_t)b * wgs) * PG_NT + threadIdx.x;
  // consecutive threads: a token's units, all heads of it, then the next token: as the cache lies
  uint32_t at = first / unit_h, in = first - at * unit_h;
  for (; at < n; at += stride_t, in += stride_in) {
    if (in >= unit_h) {
      in -= unit_h;
      if (++at >= n) break;
    }
    const int t = (int)at, h = (int)(in / units), c = (int)(in - h * units);
    const int j = t >> shift, entry = t & (C.page_size - 1);
    const int page = t < kv && j < R.table_width ? R.block_table[(int64_t)b * R.table_pitch + j] : -1;
    const bool there = page >= 0 && page < C.n_pages;
    if (COPY && entry == 0 && in == 0) O.table[(int64_t)b * copied + j] = there ? (int)page0 + j : -1;
    if (COPY && !there) continue;
    const int64_t to = ((COPY ? page0 * C.page_size * O.s_t : b * O.s_b) + h * O.s_h + t * O.s_t + (int64_t)c * E) * OS;
    char *ko = (char*)O.k + to, *vo = (char*)O.v + to;
    const char* kp = (const char*)C.k + (page * C.ks_p + entry * C.ks_t + h * C.ks_h + c * E) * CS;
    const char* vp = (const char*)C.v + (page * C.vs_p + entry * C.vs_t + h * C.vs_h + c * E) * CS;
    if constexpr (CT == SAH_E4M3) {
      uint2 k = make_uint2(0, 0), v = k;
      float ks = 1.f, vs = 1.f;
      if (there) {
        const int64_t s = ((int64_t)page * C.Hkv + h) * C.page_size + entry;
        const uint32_t k_byte = C.k_scales[s], v_byte = C.v_scales[s];
        k = *(const uint2*)kp;
        v = *(const uint2*)vp;
        ks = pg_scale(k_byte);
        vs = pg_scale(v_byte);
        if constexpr (COPY && OT == SAH_F16) lost = lost || pg_none_of_f16(k, k_byte) || pg_none_of_f16(v, v_byte);
      }
      pg_put8<OT, !COPY>(ko, k, ks);
      pg_put8<OT, !COPY>(vo, v, vs);
    } else {
      sah_u4 k = {0, 0, 0, 0}, v = k;
      if (there) {
        k = *(const sah_u4*)kp;
        v = *(const sah_u4*)vp;
      }
      pg_put16<!COPY>(ko, k);
      pg_put16<!COPY>(vo, v);
    }
  }
  if constexpr (COPY) {
    if (!O.lost) return;
    const int any = __syncthreads_or(lost);
    if (threadIdx.x == 0) O.lost[blockIdx.x] = any != 0;
  }
}

// One workgroup: how many pages each request needs, then where each one's begin (4.5 us for 64 requests, nearly all of it the launch and two readings).
__global__ __launch_bounds__(PG_NT) void k_page_place(sah_page_requests R, int page_size, int width, int64_t room, int32_t* first, int32_t* lens) {
  __shared__ int64_t s_sum[2][PG_NT / SAH_WAVE];
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id(), shift = 31 - __builtin_clz(page_size), most = R.table_width << shift;
  auto need = [&](int b, int& kv) -> int {  // pages; 0 also for requests without a row
    kv = 0;
    if (b >= R.n_requests) return 0;
    const int begin = R.cu_new[b], end = R.cu_new[b + 1];
    if ((begin > 0 ? begin : 0) >= (end < R.n_tokens ? end : R.n_tokens)) return 0;
    kv = R.kv_lens[b];
    const int held = kv < 0 ? 0 : (kv < most ? kv : most);
    return (held >> shift) + ((held & (page_size - 1)) != 0);
  };
  int turn = 0;
  auto before = [&](int64_t v, int64_t& all) -> int64_t {
    const int64_t incl = (int64_t)sah_wave_incl_scan_u64((uint64_t)v);
    if (lane == SAH_WAVE - 1) s_sum[turn][wave] = incl;
    __syncthreads();
    int64_t sum = incl - v;
    all = 0;
#pragma unroll
    for (int i = 0; i < PG_NT / SAH_WAVE; ++i) {
      sum += i < wave ? s_sum[turn][i] : 0;
      all += s_sum[turn][i];
    }
    turn ^= 1;  // (the sums of the one before may still be read)
    return sum;
  };
  int64_t total = 0, run = 0, all;
  int kv;
  bool more = false;
  for (int b = threadIdx.x; b < R.n_requests; b += PG_NT) {
    const int n = need(b, kv);
    total += n;
    more |= n > width;
  }
  (void)before(total, total);
  const bool fits = !__syncthreads_or(more) && total <= room;
  for (int b0 = 0; b0 < R.n_requests; b0 += PG_NT) {
    const int b = b0 + (int)threadIdx.x, n = need(b, kv);
    const int64_t at = run + before(n, all);
    if (b < R.n_requests) {
      first[b] = fits ? (int)at : -1;
      lens[b] = fits ? kv : 0;
    }
    run += all;
  }
}

// ---------------------------------------------------------------------------
// bounds: a wave has every n_waves-th of the pages that a request has filled, for one key head
// The chain of reads bounds it (lengths, table, four rows of a page and group of lanes at once): 1024 pages of 16 8-bit tokens, 8 heads, 21 MB, 11.7 us;
// 64 answers of which few fill a page 3.9 us. (8192 waves 11.3 and 4.8, 16384 13.2 and 5.7.)
// ---------------------------------------------------------------------------
// (a NaN is kept: comparisons with it are false)
__device__ __forceinline__ float pg_lower(float a, float b) { return b < a || b != b ? b : a; }
__device__ __forceinline__ float pg_upper(float a, float b) { return b > a || b != b ? b : a; }
// what the lanes l and l ^ 16 hold, to both of them
__device__ __forceinline__ void pg_swap16(float v, float& a, float& b) {
#if defined(__HIP_DEVICE_COMPILE__)
  const auto r = __builtin_amdgcn_permlane16_swap(sah_float_to_bits(v), sah_float_to_bits(v), false, false);
  a = sah_bits_to_float(r[0]);
  b = sah_bits_to_float(r[1]);
#else
  a = b = v;
#endif
}
template <int T>
__global__ __launch_bounds__(PG_NT) void k_page_bounds(sah_page_bounds_args P, int n_waves) {
  sah_touch_kernargs<sizeof(sah_page_bounds_args) + 4>();
  const sah_page_cache& C = P.cache;
  const sah_page_requests& R = P.requests;
  constexpr int NW = PG_NT / SAH_WAVE, E = 8;
  constexpr int BT = T == SAH_E4M3 ? SAH_BF16 : T;
  const int lane = threadIdx.x & (SAH_WAVE - 1), l16 = lane & 15, g = lane >> 4, wave = sah_wave_id();
  // key heads of a page next to each other
  const int64_t item = (int64_t)blockIdx.x * NW + wave, row = item / C.Hkv;
  const int h = (int)(item - row * C.Hkv), b = (int)(row / n_waves), turn = (int)(row - (int64_t)b * n_waves);
  if (b >= R.n_requests) return;
  const int shift = 31 - __builtin_clz(C.page_size), most = R.table_width << shift;
  const int given = R.kv_lens[b];
  const int64_t fresh = (int64_t)R.cu_new[b + 1] - R.cu_new[b];
  const int kv = given < 0 ? 0 : (given < most ? given : most);
  const int64_t before = (int64_t)given - (fresh > 0 ? fresh : 0);
  const int first = before <= 0 ? 0 : (before < kv ? (int)before : kv) >> shift, end = fresh > 0 ? kv >> shift : 0;
  for (int j = first + turn; j < end; j += n_waves) {
    const int64_t pg = R.block_table[(int64_t)b * R.table_pitch + j];
    if (pg < 0 || pg >= C.n_pages) continue;
    for (int d0 = 0; d0 < C.D; d0 += 16 * E) {  // 16 lanes' dims at a time
      const int d = d0 + l16 * E;
      const bool on = d < C.D;
      float lo[E], hi[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        lo[e] = INFINITY;
        hi[e] = -INFINITY;
      }
      constexpr int U = 4;
      for (int i0 = g; i0 < C.page_size; i0 += 4 * U) {  // four rows requested at once; behind the last one it is taken again, which changes nothing
        sah_u4 raw[U][T == SAH_F32 ? 2 : 1];
        float scale[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t i = i0 + 4 * u < C.page_size ? i0 + 4 * u : i0;
          const char* from = (const char*)C.k + (pg * C.ks_p + i * C.ks_t + h * C.ks_h + (on ? d : 0)) * pg_size(T);
          if constexpr (T == SAH_E4M3) {
            const uint2 w = *(const uint2*)from;
            raw[u][0] = sah_u4{w.x, w.y, 0, 0};
            scale[u] = pg_scale(C.k_scales[(pg * C.Hkv + h) * C.page_size + i]);
          } else {
#pragma unroll
            for (int k = 0; k < (T == SAH_F32 ? 2 : 1); ++k) raw[u][k] = ((const sah_u4*)from)[k];
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float x[E];
          if constexpr (T == SAH_E4M3) {
            float a[4], b[4];
            pg_widen4(raw[u][0].x, scale[u], a);
            pg_widen4(raw[u][0].y, scale[u], b);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = a[e];
              x[4 + e] = b[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              if constexpr (T == SAH_F32) x[e] = sah_bits_to_float(raw[u][e / 4][e % 4]);
              else if constexpr (T == SAH_BF16) x[e] = sah_bits_to_float(e % 2 ? raw[u][0][e / 2] & 0xffff0000u : raw[u][0][e / 2] << 16);
              else x[e] = sah_f16_to_float((uint16_t)(raw[u][0][e / 2] >> (16 * (e % 2))));
            }
          }
#pragma unroll
          for (int e = 0; e < E; ++e) {
            lo[e] = pg_lower(lo[e], x[e]);
            hi[e] = pg_upper(hi[e], x[e]);
          }
        }
      }
      // the four groups' rows: lanes l, l + 16, l + 32 and l + 48
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float a, b;
        pg_swap16(lo[e], a, b);
        lo[e] = pg_lower(a, b);
        pg_swap16(hi[e], a, b);
        hi[e] = pg_upper(a, b);
        uint32_t c, f;
        sah_half_both(sah_float_to_bits(lo[e]), c, f);
        lo[e] = pg_lower(sah_bits_to_float(c), sah_bits_to_float(f));
        sah_half_both(sah_float_to_bits(hi[e]), c, f);
        hi[e] = pg_upper(sah_bits_to_float(c), sah_bits_to_float(f));
      }
      if (!on || g > 1) continue;
      char* to = (char*)P.bounds + (((pg * C.Hkv + h) * 2 + g) * C.D + d) * pg_size(BT);
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = g ? hi[e] : lo[e];
      if constexpr (BT == SAH_F32) {
        ((float4*)to)[0] = make_float4(y[0], y[1], y[2], y[3]);
        ((float4*)to)[1] = make_float4(y[4], y[5], y[6], y[7]);
      } else {
        *(uint4*)to = make_uint4(sah_pack2_hw<BT>(y[0], y[1]), sah_pack2_hw<BT>(y[2], y[3]), sah_pack2_hw<BT>(y[4], y[5]), sah_pack2_hw<BT>(y[6], y[7]));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// select: a 64-bit key per candidate (larger: rather taken), then the largest of a row
// The sum over heads of max(q a, q b) with a <= b, both finite, is Q+ . b + Q- . a, Q+ (Q-) the sum of the heads' positive (negative) elements: the heads
// share one reading of the bounds and one pair of products (pages of infinite bounds: pg_score_again). In fp64, in which rounding decides between almost equal
// scores alone; fp32 is no faster (72 us against 70): reading the bounds is what it costs. 64 answers of 1K to 32K keys in pages of 16, 8 heads: 277 MB of bf16 bounds, 62 us, 4.5 TB/s; they are read past the caches, which
// they would go through once (71 us). All heads of a page by one wave 97 us, smallest and largest by neighbouring lanes 80.
// ---------------------------------------------------------------------------
#define PG_ALWAYS ~0ull        // pages that are taken whatever they score
#define PG_FIRST (~0ull - 1)   // scores that are not finite
#define PG_WAVE_PAGES 32       // pages that a wave scores at once
#define PG_SCORE_WGS 1024      // workgroups of a call, about: what the card holds at once

__device__ __forceinline__ uint64_t pg_key(double score) {  // never 0
  if (!(score - score == 0.0)) return PG_FIRST;
  const uint64_t u = __builtin_bit_cast(uint64_t, score + 0.0);  // (-0 + 0 is 0)
  return u >> 63 ? ~u : u | 1ull << 63;
}
template <int CTRL>
__device__ __forceinline__ double pg_dpp(double v) {
  return __builtin_bit_cast(double, sah_dpp_u64<CTRL, 0xF, true>(__builtin_bit_cast(uint64_t, v)));
}

// N elements (8; of fp32 also 4, of 16-bit types 4 at 8-byte addresses)
template <int T, int N>
__device__ __forceinline__ void pg_load_some(const void* p, int64_t i, float (&o)[8]) {
  if constexpr (N == 8) {
    sah_load8<T>(p, i, o);
  } else if constexpr (T == SAH_F32) {
    const float4 f = *(const float4*)((const float*)p + i);
    o[0] = f.x; o[1] = f.y; o[2] = f.z; o[3] = f.w;
  } else {
    const uint2 u = *(const uint2*)((const uint16_t*)p + i);
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      o[2 * k] = T == SAH_BF16 ? sah_bits_to_float(w[k] << 16) : sah_f16_to_float((uint16_t)w[k]);
      o[2 * k + 1] = T == SAH_BF16 ? sah_bits_to_float(w[k] & 0xffff0000u) : sah_f16_to_float((uint16_t)(w[k] >> 16));
    }
  }
}

struct pg_select {
  sah_page_select_args a;
  int64_t row0;  // the first of the rows (token, key head) that are looked at: a call goes through them in slices that its workspace has room for
  int pitch;     // keys of a row
  int chunks;    // workgroups a row, which take its pages in turn
};

__device__ __forceinline__ float pg_load_as(int dtype, const void* p, int64_t i) {
  return dtype == SAH_F32 ? sah_load<SAH_F32>(p, i) : dtype == SAH_BF16 ? sah_load<SAH_BF16>(p, i) : sah_load<SAH_F16>(p, i);
}
// The score of a page by a whole wave, for those whose sum of Q+ . max + Q- . min is not finite: an infinite smallest element counts only where
// some head is not positive, a largest one where some head is not negative. Elsewhere the larger product is the other one, not 0 times infinity.
__device__ __forceinline__ double pg_score_again(const sah_page_select_args& P, int64_t t, int h, int page) {
  const int lane = threadIdx.x & (SAH_WAVE - 1), G = P.Hq / P.Hkv;
  const int64_t q = t * P.qs_t + (int64_t)h * G * P.qs_h, b = ((int64_t)page * P.Hkv + h) * 2 * P.D;
  double sum = 0.0;
#pragma unroll 1
  for (int d = lane; d < P.D; d += SAH_WAVE) {
    double up = 0.0, down = 0.0;
    bool positive = true, negative = true;  // all heads
#pragma unroll 1
    for (int i = 0; i < G; ++i) {
      const float x = pg_load_as(P.dtype, P.q, q + i * P.qs_h + d);
      up += x < 0.f ? 0.0 : (double)x;
      down += x < 0.f ? (double)x : 0.0;
      positive &= x > 0.f;
      negative &= x < 0.f;
    }
    const float lo = pg_load_as(P.bounds_dtype, P.bounds, b + d), hi = pg_load_as(P.bounds_dtype, P.bounds, b + P.D + d);
    if (!(positive && fabsf(lo) == INFINITY)) sum = fma(down, (double)lo, sum);
    if (!(negative && fabsf(hi) == INFINITY)) sum = fma(up, (double)hi, sum);
  }
#pragma unroll
  for (int i = 1; i < SAH_WAVE; i *= 2) sum += __shfl_xor(sum, i);
  return sum;
}

// BT: type of the bounds, DP: D up to 64, 128 or 256. L lanes hold a page's row of bounds, E elements of each of the two.
template <int BT, int DP>
__global__ __launch_bounds__(PG_NT, (BT == SAH_F32 || DP <= 128 ? 4 : 3)) void k_page_scores(pg_select S) {
  sah_touch_kernargs<sizeof(pg_select)>();
  const sah_page_select_args& P = S.a;
  const sah_page_requests& R = P.requests;
  constexpr int NW = PG_NT / SAH_WAVE, ES = pg_size(BT), E = 16 / ES, L = DP / E;
  constexpr int AT_ONCE = SAH_WAVE / L;                    // pages in a load instruction
  constexpr int U = PG_WAVE_PAGES / AT_ONCE < 8 ? PG_WAVE_PAGES / AT_ONCE : 8;
  const int lane = threadIdx.x & (SAH_WAVE - 1), in = lane % L, who = lane / L, wave = sah_wave_id();
  const int64_t row = blockIdx.x / S.chunks;
  const int chunk = (int)(blockIdx.x - row * S.chunks);
  const int64_t t = (S.row0 + row) / P.Hkv;
  const int h = (int)(S.row0 + row - t * P.Hkv);
  const pg_request r = pg_find_by_wave(R, P.page_size, (int)t);
  if (r.b < 0) return;
  int64_t p = r.base + t;
  if (p >= r.kv) p = r.kv - 1;
  if (p < 0) return;
  const int shift = 31 - __builtin_clz(P.page_size), n = (int)(p >> shift) + 1;
  if ((chunk * NW + wave) * PG_WAVE_PAGES >= n) return;
  // the group's queries, the positive and the negative ones of a channel added up (numbers of at most 24 bits: exact for what is not wide apart)
  const int G = P.Hq / P.Hkv;
  double up[E], down[E];
#pragma unroll
  for (int e = 0; e < E; ++e) up[e] = down[e] = 0.0;
  if (in * E < P.D) {
    const int64_t first = t * P.qs_t + (int64_t)h * G * P.qs_h + in * E;
    auto add = [&](auto type) __attribute__((always_inline)) {
      constexpr int QT = decltype(type)::value;
#pragma unroll 4
      for (int i = 0; i < G; ++i) {
        float q[8];
        pg_load_some<QT, E>(P.q, first + i * P.qs_h, q);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          up[e] += q[e] < 0.f ? 0.0 : (double)q[e];  // (NaN too)
          down[e] += q[e] < 0.f ? (double)q[e] : 0.0;
        }
      }
    };
    if (P.dtype == SAH_F32) add(std::integral_constant<int, SAH_F32>());
    else if (P.dtype == SAH_BF16) add(std::integral_constant<int, SAH_BF16>());
    else add(std::integral_constant<int, SAH_F16>());
  }
  uint64_t* keys = (uint64_t*)P.work + row * S.pitch;
  const char* base = (const char*)P.bounds + (int64_t)h * 2 * P.D * ES;
  bool odd = false;  // a score that is not finite
  for (int64_t from = (chunk * NW + wave) * PG_WAVE_PAGES; from < n; from += (int64_t)S.chunks * NW * PG_WAVE_PAGES) {
    // a lane's page
    const int j0 = (int)from, j = j0 + lane;
    const bool mine = lane < PG_WAVE_PAGES && j < n;
    int page = mine ? R.block_table[(int64_t)r.b * R.table_pitch + j] : -1;
    if (page >= P.n_pages) page = -1;
    const bool always = j < P.sink_pages || j >= n - P.window_pages;
    for (int i0 = 0; i0 < PG_WAVE_PAGES; i0 += U * AT_ONCE) {
      if (j0 + i0 >= n) break;
      sah_u4 lo[U], hi[U];
      int at[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        at[i] = __shfl(always ? -1 : page, i0 + i * AT_ONCE + who);
        lo[i] = hi[i] = sah_u4{0, 0, 0, 0};
        if (at[i] >= 0 && in * E < P.D) {
          const char* b = base + (int64_t)at[i] * P.Hkv * 2 * P.D * ES + 16 * in;
          lo[i] = __builtin_nontemporal_load((const sah_u4*)b);
          hi[i] = __builtin_nontemporal_load((const sah_u4*)(b + P.D * ES));
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const uint32_t a[4] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w}, z[4] = {hi[i].x, hi[i].y, hi[i].z, hi[i].w};
        double sum = 0.0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (BT == SAH_F32) {
            sum = fma(down[w], (double)sah_bits_to_float(a[w]), sum);
            sum = fma(up[w], (double)sah_bits_to_float(z[w]), sum);
          } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float x, y;
              if constexpr (BT == SAH_BF16) {
                x = sah_bits_to_float(half ? a[w] & 0xffff0000u : a[w] << 16);
                y = sah_bits_to_float(half ? z[w] & 0xffff0000u : z[w] << 16);
              } else {
                x = sah_f16_to_float((uint16_t)(a[w] >> (16 * half)));
                y = sah_f16_to_float((uint16_t)(z[w] >> (16 * half)));
              }
              sum = fma(down[2 * w + half], (double)x, sum);
              sum = fma(up[2 * w + half], (double)y, sum);
            }
          }
        }
        if constexpr (L >= 2) sum += pg_dpp<0xB1>(sum);
        if constexpr (L >= 4) sum += pg_dpp<0x4E>(sum);
        if constexpr (L >= 8) sum += pg_dpp<0x141>(sum);
        if constexpr (L >= 16) sum += pg_dpp<0x140>(sum);
        if constexpr (L >= 32) sum += __shfl_xor(sum, 16);
        if constexpr (L >= 64) sum += __shfl_xor(sum, 32);
        const int to = j0 + i0 + i * AT_ONCE + who;
        odd |= !(sum - sum == 0.0);
        if (in == 0 && at[i] >= 0 && to < n) keys[to] = pg_key(sum);
      }
    }
    if (mine && (always || page < 0)) keys[j] = page < 0 ? 0 : PG_ALWAYS;
    if (!__ballot(odd)) continue;
    odd = false;
    for (int i = 0; i < PG_WAVE_PAGES && j0 + i < n; ++i) {
      const int page_of = __builtin_amdgcn_readlane(always ? -1 : page, i);
      if (page_of < 0) continue;
      const double sum = pg_score_again(P, t, h, page_of);
      if (lane == 0) keys[j0 + i] = pg_key(sum);
    }
  }
}

// Sum of one number per thread before it, across the workgroup, and of all; `wsum`: PG_NT / 64 words that no other call uses.
__device__ __forceinline__ int pg_before(int v, int* wsum, int& all) {
  constexpr int NW = PG_NT / SAH_WAVE;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const int incl = sah_wave_incl_scan(v);
  if (lane == SAH_WAVE - 1) wsum[wave] = incl;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    before += i < wave ? wsum[i] : 0;
    all += wsum[i];
  }
  return before + incl - v;
}
// bits that any of the wave's lanes has set (in its last lane)
__device__ __forceinline__ uint32_t pg_any_bits(uint32_t v) {
  int x = (int)v;
  x |= sah_dpp_i<0x111, 0xF, true>(x);
  x |= sah_dpp_i<0x112, 0xF, true>(x);
  x |= sah_dpp_i<0x114, 0xF, true>(x);
  x |= sah_dpp_i<0x118, 0xF, true>(x);
  x |= sah_dpp_i<0x142, 0xA, false>(x);
  x |= sah_dpp_i<0x143, 0xC, false>(x);
  return (uint32_t)x;
}

// One workgroup a row: the digit of 8 bits at which the count of the larger keys passes n_select, from the highest bit on in which the row's keys
// differ, in an LDS histogram; again inside that digit, unless its keys fit a list of one wave, which ranks them against each other.
// Then the places of what is taken, in the order of the table. A thread has neighbouring pages.
#define PG_DIGIT 8
#define PG_LIST SAH_WAVE
__global__ __launch_bounds__(PG_NT) void k_page_top(pg_select S) {
  sah_touch_kernargs<sizeof(pg_select)>();
  const sah_page_select_args& P = S.a;
  constexpr int NW = PG_NT / SAH_WAVE, KEEP = 8, BINS = 1 << PG_DIGIT, MINE = BINS / PG_NT;
  __shared__ int s_hist[BINS];
  __shared__ int s_sum[5][NW];
  __shared__ uint64_t s_ones[NW], s_zeros[NW], s_key[PG_LIST], s_border;
  __shared__ int s_at[PG_LIST], s_border_at, s_listed, s_bin, s_above, s_count;
  const int64_t row = S.row0 + blockIdx.x, t = row / P.Hkv;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const pg_request r = pg_find_by_wave(P.requests, P.page_size, (int)t);
  int64_t p = r.b < 0 ? -1 : r.base + t;
  if (p >= r.kv) p = r.kv - 1;
  const int shift = 31 - __builtin_clz(P.page_size), n = p < 0 ? 0 : (int)(p >> shift) + 1;
  int32_t* out = P.pages + row * P.n_select;
  const uint64_t* keys = (const uint64_t*)P.work + (int64_t)blockIdx.x * S.pitch;
  const int each = (n + PG_NT - 1) / PG_NT, first = (int)threadIdx.x * each;
  const bool kept = each <= KEEP;  // in registers, else read again whenever they are looked at
  uint64_t mine[KEEP];
#pragma unroll
  for (int i = 0; i < KEEP; ++i) mine[i] = kept && i < each && first + i < n ? keys[first + i] : 0;
  auto visit = [&](auto f) __attribute__((always_inline)) {
    if (kept) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (i < each) f(first + i, mine[i]);
    } else {
      for (int i = 0; i < each; ++i) f(first + i, first + i < n ? keys[first + i] : 0);
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < MINE; ++i) s_hist[(int)threadIdx.x + i * PG_NT] = 0;
    if (threadIdx.x == 0) s_listed = 0;
  };
  clear();
  // Those that are ranked (not the ones that are taken anyway: their key would hide where the others' differ), and which bits are set, and which
  // are not, in any of them
  auto ranks = [](uint64_t key) { return (key != 0) & (key != PG_ALWAYS); };
  uint64_t ones = 0, zeros = 0;
  int count = 0, fixed = 0;
  visit([&](int, uint64_t key) {
    const bool in = ranks(key);
    count += in;
    fixed += key == PG_ALWAYS;
    ones |= in ? key : 0;
    zeros |= in ? ~key : 0;
  });
  const uint32_t o0 = pg_any_bits((uint32_t)ones), o1 = pg_any_bits((uint32_t)(ones >> 32));
  const uint32_t z0 = pg_any_bits((uint32_t)zeros), z1 = pg_any_bits((uint32_t)(zeros >> 32));
  if (lane == SAH_WAVE - 1) {
    s_ones[wave] = (uint64_t)o1 << 32 | o0;
    s_zeros[wave] = (uint64_t)z1 << 32 | z0;
  }
  int total, always;
  (void)pg_before(fixed, s_sum[2], always);
  (void)pg_before(count, s_sum[0], total);
  ones = zeros = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    ones |= s_ones[i];
    zeros |= s_zeros[i];
  }
  // Taken: keys whose bits from `low` on are more than `prefix`, and `want` of the `inside` ones for which they are just that.
  int low = 64, want = total, inside = total;  // (no bits: all)
  uint64_t prefix = 0;
  auto upper = [&](uint64_t key) { return low < 64 ? key >> low : 0; };
  if (total > P.n_select - always) {
    const uint64_t differ = ones & zeros;
    low = differ ? 64 - __builtin_clzll(differ) : 0;
    prefix = upper(ones);
    want = P.n_select - always;
    int round = 0;
    while (low > 0 && inside > PG_LIST && inside > want && want) {  // (at most 8 times)
      const int width = low < PG_DIGIT ? low : PG_DIGIT, next = low - width;
      visit([&](int, uint64_t key) {
        if (ranks(key) && upper(key) == prefix) atomicAdd(&s_hist[(key >> next) & ((1u << width) - 1)], 1);
      });
      __syncthreads();
      // a thread's neighbouring digits, the largest in thread 0
      int c[MINE], sum = 0;
#pragma unroll
      for (int i = 0; i < MINE; ++i) sum += c[i] = s_hist[BINS - 1 - MINE * (int)threadIdx.x - i];
      int all;
      int above = pg_before(sum, s_sum[1 + (round++ & 1)], all);  // (those of the round before may still be read)
      if (above < want && want <= above + sum) {
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          if (above < want && want <= above + c[i]) {
            s_bin = BINS - 1 - MINE * (int)threadIdx.x - i;
            s_above = above;
            s_count = c[i];
          }
          above += c[i];
        }
      }
      clear();          // (all have read their digits: the wait above)
      __syncthreads();
      want -= s_above;
      inside = s_count;
      prefix = (low < 64 ? prefix << width : 0) | (uint64_t)s_bin;
      low = next;
    }
  }
  // the last one taken, by key and, of equal keys, place
  uint64_t border = low < 64 ? (prefix << low) - 1 : 0;  // (all of the inside ones: what lies above their smallest number less one)
  int border_at = -1;
  if (want == 0) border = PG_ALWAYS - 1;
  else if (want < inside && low > 0) {  // uniform: a list of at most PG_LIST
    visit([&](int j, uint64_t key) {
      if (!ranks(key) || upper(key) != prefix) return;
      const int i = atomicAdd(&s_listed, 1);
      s_key[i] = key;
      s_at[i] = j;
    });
    __syncthreads();
    if (wave == 0) {
      const uint64_t key = s_key[lane];  // (lanes beyond the list hold nobody's)
      const int at = s_at[lane];
      int ahead = 0;
#pragma unroll 4
      for (int i = 0; i < inside; ++i) ahead += (s_key[i] > key) | ((s_key[i] == key) & (s_at[i] < at));
      if (lane < inside && ahead == want - 1) {
        s_border = key;
        s_border_at = at;
      }
    }
    __syncthreads();
    border = s_border;
    border_at = s_border_at;
  }
  int all, taken;
  if (low == 0 && want && want < inside) {  // equal keys, more than the list holds: the first `want` of them
    int n_larger = 0, n_equal = 0;
    visit([&](int, uint64_t key) {
      n_larger += key > prefix;
      n_equal += key == prefix;
    });
    int larger = pg_before(n_larger, s_sum[3], all);
    taken = all + want;
    int ranked = pg_before(n_equal, s_sum[4], all);
    visit([&](int j, uint64_t key) {
      if (key < prefix) return;
      if (key > prefix || ranked < want) out[larger + (ranked < want ? ranked : want)] = j;
      larger += key > prefix;
      ranked += key == prefix;
    });
  } else {
    auto take = [&](int j, uint64_t key) { return (key > border) | ((key == border) & (j <= border_at)); };
    int n_taken = 0;
    visit([&](int j, uint64_t key) { n_taken += take(j, key); });
    int at = pg_before(n_taken, s_sum[3], taken);
    visit([&](int j, uint64_t key) {
      if (take(j, key)) out[at++] = j;
    });
  }
  for (int i = taken + (int)threadIdx.x; i < P.n_select; i += PG_NT) out[i] = -1;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
extern "C" int sah_page_store(const sah_page_store_args* given) {
  static const char* what = "sah_page_store";
  if (!given) return sah_fail(SAH_ENULL, "sah_page_store: args is NULL");
  sah_page_store_args own = *given;
  sah_page_store_args* a = &own;
  sah_page_cache& c = a->cache;
  if (int rc = pg_check_cache(c, true, what)) return rc;
  if (c.dtype != SAH_E4M3) return sah_fail(SAH_EDTYPE, "sah_page_store: the cache's dtype is %d, not SAH_E4M3", c.dtype);
  if (a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16) return sah_fail(SAH_EDTYPE, "sah_page_store: dtype %d", a->dtype);
  if (a->n_tokens < 0) return sah_fail(SAH_EINVAL, "sah_page_store: n_tokens is negative");
  if (a->n_tokens == 0) return SAH_OK;
  if (!a->k || !a->v || !a->slot_map) return sah_fail(SAH_ENULL, "sah_page_store: NULL pointer");
  if (a->n_tokens == 1) a->ks_t = a->vs_t = 0;
  if (c.Hkv == 1) a->ks_h = a->vs_h = 0;
  const int es = pg_size(a->dtype);
  if (((uint64_t)a->k | (uint64_t)a->v | (uint64_t)(es * (a->ks_t | a->ks_h | a->vs_t | a->vs_h))) % 16)
    return sah_fail(SAH_EINVAL, "sah_page_store: addresses and strides must be multiples of 16 bytes");
  if (!sah_rows_apart<3>(c.D, {c.ks_p, c.ks_t, c.ks_h}, {c.n_pages, c.page_size, c.Hkv}) ||
      !sah_rows_apart<3>(c.D, {c.vs_p, c.vs_t, c.vs_h}, {c.n_pages, c.page_size, c.Hkv}))
    return sah_fail(SAH_EINVAL, "sah_page_store: rows of a cache overlap");
  const int64_t wgs = ((int64_t)a->n_tokens * c.Hkv + PG_NT / 16 - 1) / (PG_NT / 16);
  if (wgs > 0x7fffffff) return sah_fail(SAH_ESHAPE, "sah_page_store: too many rows");
  sah_timed timed("k_page_store", a->stream);
  const dim3 grid((unsigned)wgs);
  hipStream_t st = (hipStream_t)a->stream;
  if (a->dtype == SAH_F32) hipLaunchKernelGGL(k_page_store<SAH_F32>, grid, dim3(PG_NT), 0, st, *a);
  else if (a->dtype == SAH_BF16) hipLaunchKernelGGL(k_page_store<SAH_BF16>, grid, dim3(PG_NT), 0, st, *a);
  else hipLaunchKernelGGL(k_page_store<SAH_F16>, grid, dim3(PG_NT), 0, st, *a);
  return sah_launch_status(what);
}

int64_t pg_load_workgroups(const sah_page_cache& c, const sah_page_requests& r, int length) {
  const int64_t units = (int64_t)c.D / (c.dtype == SAH_E4M3 ? 8 : 16 / pg_size(c.dtype)) * c.Hkv * length, room = PG_LOAD_WGS / r.n_requests;
  int64_t wgs = (units + PG_NT - 1) / PG_NT;
  if (wgs > INT32_MAX / r.n_requests) return 0;
  if (wgs > room) wgs = room > 1 ? room : 1;
  return wgs * r.n_requests;
}
// (also what the attention over chunks makes its copy with)
int pg_load(const sah_page_cache& c, const sah_page_requests& r, int dtype, const pg_load_out& out, void* stream, const char* what) {
  const int64_t all = pg_load_workgroups(c, r, out.length), wgs = all / r.n_requests;
  if (!all) return sah_fail(SAH_ESHAPE, "%s: too many elements", what);
  sah_timed timed("k_page_load", stream);
  const dim3 grid((unsigned)all);
  hipStream_t st = (hipStream_t)stream;
  if (c.dtype == SAH_F32) hipLaunchKernelGGL((k_page_load<SAH_F32, SAH_F32, false>), grid, dim3(PG_NT), 0, st, c, r, out, (int)wgs);
  else if (c.dtype != SAH_E4M3) hipLaunchKernelGGL((k_page_load<SAH_BF16, SAH_BF16, false>), grid, dim3(PG_NT), 0, st, c, r, out, (int)wgs);
  else if (dtype == SAH_F32) hipLaunchKernelGGL((k_page_load<SAH_E4M3, SAH_F32, false>), grid, dim3(PG_NT), 0, st, c, r, out, (int)wgs);
  else if (out.table && dtype == SAH_BF16) hipLaunchKernelGGL((k_page_load<SAH_E4M3, SAH_BF16, true>), grid, dim3(PG_NT), 0, st, c, r, out, (int)wgs);
  else if (out.table) hipLaunchKernelGGL((k_page_load<SAH_E4M3, SAH_F16, true>), grid, dim3(PG_NT), 0, st, c, r, out, (int)wgs);
  else if (dtype == SAH_BF16) hipLaunchKernelGGL((k_page_load<SAH_E4M3, SAH_BF16, false>), grid, dim3(PG_NT), 0, st, c, r, out, (int)wgs);
  else hipLaunchKernelGGL((k_page_load<SAH_E4M3, SAH_F16, false>), grid, dim3(PG_NT), 0, st, c, r, out, (int)wgs);
  return sah_launch_status(what);
}

int pg_place(const sah_page_requests& r, int page_size, int width, int64_t room, int32_t* first, int32_t* lens, void* stream, const char* what) {
  sah_timed timed("k_page_place", stream);
  hipLaunchKernelGGL(k_page_place, dim3(1), dim3(PG_NT), 0, (hipStream_t)stream, r, page_size, width, room, first, lens);
  return sah_launch_status(what);
}

extern "C" int sah_page_load(const sah_page_load_args* given) {
  static const char* what = "sah_page_load";
  if (!given) return sah_fail(SAH_ENULL, "sah_page_load: args is NULL");
  sah_page_load_args own = *given;
  sah_page_load_args* a = &own;
  sah_page_cache& c = a->cache;
  if (int rc = pg_check_cache(c, true, what)) return rc;
  if (int rc = pg_check_requests(a->requests, c.page_size, false, what)) return rc;
  if (c.dtype == SAH_E4M3 ? a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16 : a->dtype != c.dtype)
    return sah_fail(SAH_EDTYPE, "sah_page_load: dtype %d of a cache of dtype %d", a->dtype, c.dtype);
  if (a->length < 0) return sah_fail(SAH_EINVAL, "sah_page_load: length is negative");
  if (a->length == 0) return SAH_OK;
  if (!a->k_out || !a->v_out) return sah_fail(SAH_ENULL, "sah_page_load: NULL pointer");
  if (((uint64_t)a->k_out | (uint64_t)a->v_out) % 16) return sah_fail(SAH_EINVAL, "sah_page_load: addresses must be multiples of 16 bytes");
  if (!pg_load_workgroups(c, a->requests, a->length)) return sah_fail(SAH_ESHAPE, "sah_page_load: too many elements");
  const int64_t row = c.D, head = row * a->length;
  const sah_span k = pg_span(a->k_out, a->requests.n_requests, c.Hkv, head, pg_size(a->dtype)), v = pg_span(a->v_out, a->requests.n_requests, c.Hkv, head, pg_size(a->dtype));
  if (sah_meet(k, v) || pg_on_cache(k, c) || pg_on_cache(v, c) || pg_on_requests(k, a->requests, false) || pg_on_requests(v, a->requests, false))
    return sah_fail(SAH_EINVAL, "sah_page_load: k_out or v_out shares memory with the other, the cache, the table or the lengths");
  return pg_load(c, a->requests, a->dtype, pg_load_out{a->k_out, a->v_out, head * c.Hkv, head, row, a->length, nullptr, nullptr, nullptr}, a->stream, what);
}

extern "C" int sah_page_bounds(const sah_page_bounds_args* given) {
  static const char* what = "sah_page_bounds";
  if (!given) return sah_fail(SAH_ENULL, "sah_page_bounds: args is NULL");
  sah_page_bounds_args own = *given;
  sah_page_bounds_args* a = &own;
  sah_page_cache& c = a->cache;
  if (int rc = pg_check_cache(c, false, what)) return rc;
  if (int rc = pg_check_requests(a->requests, c.page_size, true, what)) return rc;
  if (!a->bounds) return sah_fail(SAH_ENULL, "sah_page_bounds: NULL pointer");
  if ((uint64_t)a->bounds % 16) return sah_fail(SAH_EINVAL, "sah_page_bounds: addresses must be multiples of 16 bytes");
  const sah_span bounds = pg_span(a->bounds, c.n_pages, c.Hkv, 2 * c.D, c.dtype == SAH_E4M3 ? 2 : pg_size(c.dtype));
  if (pg_on_cache(bounds, c) || pg_on_requests(bounds, a->requests, true))
    return sah_fail(SAH_EINVAL, "sah_page_bounds: bounds share memory with the keys, the table or the lengths");
  // Enough waves for the card where few requests have filled many pages; each of many requests' fills few.
  const int64_t rows = (int64_t)a->requests.n_requests * c.Hkv;
  int64_t n_waves = PG_BOUND_WAVES / rows;
  n_waves = n_waves < 1 ? 1 : (n_waves < a->requests.table_width ? n_waves : a->requests.table_width);
  const int64_t wgs = (rows * n_waves + PG_NT / SAH_WAVE - 1) / (PG_NT / SAH_WAVE);
  if (wgs > 0x7fffffff) return sah_fail(SAH_ESHAPE, "sah_page_bounds: too many rows");
  sah_timed timed("k_page_bounds", a->stream);
  const dim3 grid((unsigned)wgs);
  hipStream_t st = (hipStream_t)a->stream;
  if (c.dtype == SAH_F32) hipLaunchKernelGGL(k_page_bounds<SAH_F32>, grid, dim3(PG_NT), 0, st, *a, (int)n_waves);
  else if (c.dtype == SAH_BF16) hipLaunchKernelGGL(k_page_bounds<SAH_BF16>, grid, dim3(PG_NT), 0, st, *a, (int)n_waves);
  else if (c.dtype == SAH_F16) hipLaunchKernelGGL(k_page_bounds<SAH_F16>, grid, dim3(PG_NT), 0, st, *a, (int)n_waves);
  else hipLaunchKernelGGL(k_page_bounds<SAH_E4M3>, grid, dim3(PG_NT), 0, st, *a, (int)n_waves);
  return sah_launch_status(what);
}

// Rows of a slice: all of them up to 256 MiB of keys (2048 tokens, 8 key heads, tables of 131072 tokens in pages of
// 16: 1 GiB; in slices 16.1 ms instead of 18.7 over 130000 keys, 0.97 instead of 0.91 over 20000).
#define PG_SELECT_BYTES (1 << 28)
static int64_t pg_select_rows(const sah_page_select_args* a) {
  const int64_t rows = (int64_t)a->requests.n_tokens * a->Hkv, room = PG_SELECT_BYTES / ((int64_t)a->requests.table_width * 8);
  return rows < room ? rows : room > 1 ? room : 1;
}
extern "C" int64_t sah_page_select_work_bytes(const sah_page_select_args* a) {
  if (!a || a->requests.n_tokens <= 0 || a->Hkv <= 0 || a->requests.table_width <= 0) return 0;
  return pg_select_rows(a) * a->requests.table_width * 8;
}

extern "C" int sah_page_select(const sah_page_select_args* given) {
  if (!given) return sah_fail(SAH_ENULL, "sah_page_select: args is NULL");
  sah_page_select_args own = *given;
  sah_page_select_args* a = &own;
  if (a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16) return sah_fail(SAH_EDTYPE, "sah_page_select: dtype %d", a->dtype);
  if (a->bounds_dtype != SAH_F32 && a->bounds_dtype != SAH_BF16 && a->bounds_dtype != SAH_F16)
    return sah_fail(SAH_EDTYPE, "sah_page_select: bounds of dtype %d", a->bounds_dtype);
  if (a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->n_pages <= 0 || a->max_context < 0)
    return sah_fail(SAH_EINVAL, "sah_page_select: bad sizes (heads %d / %d, n_pages %d, max_context %d)", a->Hq, a->Hkv, a->n_pages, a->max_context);
  if (a->D <= 0 || a->D % 8 || a->D > PG_MAX_D) return sah_fail(SAH_ESHAPE, "sah_page_select: head_dim %d is not a multiple of 8 up to 256", a->D);
  if (a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return sah_fail(SAH_ESHAPE, "sah_page_select: page_size %d is not a power of two", a->page_size);
  if (a->sink_pages < 0 || a->window_pages < 1 || (int64_t)a->sink_pages + a->window_pages > a->n_select)
    return sah_fail(SAH_EINVAL, "sah_page_select: %d first and %d last pages of %d", a->sink_pages, a->window_pages, a->n_select);
  if (int rc = pg_check_requests(a->requests, a->page_size, true, "sah_page_select")) return rc;
  if (a->requests.n_tokens == 0) return SAH_OK;
  if (!a->q || !a->bounds || !a->pages) return sah_fail(SAH_ENULL, "sah_page_select: NULL pointer");
  if (!a->work || a->work_bytes < sah_page_select_work_bytes(a) || (uint64_t)a->work % 16) return sah_fail(SAH_ECAPACITY, "sah_page_select: work is too small");
  if (a->requests.n_tokens == 1) a->qs_t = 0;
  if (a->Hq == 1) a->qs_h = 0;
  if (((uint64_t)a->q | (uint64_t)a->bounds | (uint64_t)(pg_size(a->dtype) * (a->qs_t | a->qs_h))) % 16)
    return sah_fail(SAH_EINVAL, "sah_page_select: addresses and strides must be multiples of 16 bytes");
  const int64_t rows = (int64_t)a->requests.n_tokens * a->Hkv;
  if (rows > 0x7fffffff) return sah_fail(SAH_ESHAPE, "sah_page_select: too many rows");
  const sah_span pages = pg_span(a->pages, rows, a->n_select, 1, 4);
  if (sah_meet(pages, sah_span_of<2>(a->q, pg_size(a->dtype), a->D, {a->qs_t, a->qs_h}, {a->requests.n_tokens, a->Hq})) ||
      sah_meet(pages, pg_span(a->bounds, a->n_pages, a->Hkv, 2 * a->D, pg_size(a->bounds_dtype))) || pg_on_requests(pages, a->requests, true))
    return sah_fail(SAH_EINVAL, "sah_page_select: pages share memory with the queries, the bounds, the table or the lengths");
  const int per = PG_WAVE_PAGES * (PG_NT / SAH_WAVE), width = a->requests.table_width;
  const int64_t hint = ((int64_t)a->max_context + a->page_size - 1) / a->page_size;
  const int usual = hint > 0 && hint < width ? (int)hint : width;  // pages of the longest request, by what the caller says
  const int64_t most = pg_select_rows(a), room = PG_SCORE_WGS / most > 1 ? PG_SCORE_WGS / most : 1;
  int64_t chunks = (usual + per - 1) / per;
  if (chunks > room) chunks = room;
  hipStream_t st = (hipStream_t)a->stream;
  for (int64_t row0 = 0; row0 < rows; row0 += most) {
    const int64_t n = rows - row0 < most ? rows - row0 : most;
    const pg_select s{*a, row0, width, (int)chunks};
    {
      sah_timed timed("k_page_scores", a->stream);
      const dim3 grid((unsigned)(n * chunks));
      const int dp = a->D <= 64 ? 64 : a->D <= 128 ? 128 : 256;
#define PG_CASE(bt, d) if (a->bounds_dtype == bt && dp == d) hipLaunchKernelGGL((k_page_scores<bt, d>), grid, dim3(PG_NT), 0, st, s);
      PG_CASE(SAH_F32, 64) PG_CASE(SAH_F32, 128) PG_CASE(SAH_F32, 256)
      PG_CASE(SAH_BF16, 64) PG_CASE(SAH_BF16, 128) PG_CASE(SAH_BF16, 256)
      PG_CASE(SAH_F16, 64) PG_CASE(SAH_F16, 128) PG_CASE(SAH_F16, 256)
#undef PG_CASE
      if (int rc = sah_launch_status("sah_page_select")) return rc;
    }
    sah_timed timed("k_page_top", a->stream);
    hipLaunchKernelGGL(k_page_top, dim3((unsigned)n), dim3(PG_NT), 0, st, s);
    if (int rc = sah_launch_status("sah_page_select(top)")) return rc;
  }
  return SAH_OK;
}
