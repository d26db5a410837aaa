// A key-value cache in pages: places for new tokens, pages given back, keys and values written to their slots.
#include "sah_common.h"
#include "../../include/sah_serve.h"

#define PG_NT 1024
#define PG_MAX_REQ 4096   // records of all requests fit into 48 KB of LDS
#define PG_REFUSED INT32_MIN

// Exclusive scan of one 64-bit number per thread across PG_NT threads; *total: the sum. All threads call.
__device__ __forceinline__ int64_t pg_scan(int64_t v, int64_t* wsum, int64_t* total) {
  constexpr int NW = PG_NT / SAH_WAVE;
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const int64_t incl = (int64_t)sah_wave_incl_scan_u64((uint64_t)v);
  __syncthreads();  // wsum may still be read from the call before
  if (lane == SAH_WAVE - 1) wsum[wave] = incl;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const int64_t s = wsum[i];
    before += i < wave ? s : 0;
    all += s;
  }
  *total = all;
  return before + incl - v;
}

// Row t's request among `n` whose rows end at s_end[0 .. n) (not falling): the first whose end lies behind t.
__device__ __forceinline__ int pg_request_of(const int* s_end, int n, int t) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s_end[mid] > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// Places of rows t = first, first + step, ... A token that opens a page (every new page has one) writes the page's entry of
// the table. s_rec: the request's length before the step, and the place in the free list of its first new page.
__device__ __forceinline__ void pg_place(const sah_paged_assign_args& P, const int* s_end, const int2* s_rec, int first, int step) {
  for (int t = first; t < P.n_tokens; t += step) {
    const int b = pg_request_of(s_end, P.n_requests, t);
    int64_t slot = -1;
    int pos = 0;
    if (b < P.n_requests) {
      const int2 rec = s_rec[b];
      pos = (int)((uint32_t)rec.x + (uint32_t)(t - (b ? s_end[b - 1] : 0)));
      if (rec.y != PG_REFUSED) {
        const int j = pos / P.page_size, entry = pos - j * P.page_size;
        const int had = (int)(((int64_t)rec.x + P.page_size - 1) / P.page_size);
        int32_t* te = P.block_table + (int64_t)b * P.table_pitch + j;
        int page;
        if (j >= had) {
          page = P.free_pages[rec.y - (j - had)];
          if (entry == 0) *te = page;
        } else {
          page = *te;
        }
        slot = page < 0 ? -1 : (int64_t)page * P.page_size + entry;
      }
    }
    P.slot_map[t] = slot;
    P.positions[t] = pos;
  }
}

// One workgroup goes over the requests: who is granted depends on all requests before, and their running sums are two scans of up to 4096
// numbers, latency and nothing else (64 requests: 5.4 us, of which a launch is 2). With ALL it also places the tokens, else it leaves
// the records for k_paged_place. One kernel up to 1024 tokens, one a thread (64 requests of 16: 6.8 us, 8.0 in two); the second kernel
// from there on (4096 tokens: 10.1 us in one, 8.4 in two; 32768: 41 and 8.5).
template <bool ALL>
__global__ __launch_bounds__(PG_NT) void k_paged_assign(sah_paged_assign_args P) {
  sah_touch_kernargs<sizeof(sah_paged_assign_args)>();
  SAH_DYNAMIC_LDS(s_dyn);
  __shared__ int64_t s_sum[PG_NT / SAH_WAVE];
  int2* s_rec = (int2*)s_dyn;
  int* s_end = (int*)(s_rec + P.n_requests);
  int64_t count = *P.free_count;
  if (count > P.n_pages) count = P.n_pages;
  if (count < 0) count = 0;
  int64_t rows = 0, pages = 0;   // of the requests before this round's
  int taken = 0;                 // this thread's last granted page
  for (int b0 = 0; b0 < P.n_requests; b0 += PG_NT) {
    const int b = b0 + threadIdx.x;
    const bool live = b < P.n_requests;
    const int given = live ? P.new_lens[b] : 0;
    const int64_t fresh = given > 0 ? given : 0, len = live ? P.lens[b] : 0;
    int64_t all;
    const int64_t begin = rows + pg_scan(fresh, s_sum, &all);
    rows += all;
    const int64_t had = (len + P.page_size - 1) / P.page_size, has = (len + fresh + P.page_size - 1) / P.page_size;
    const bool fits = live && len >= 0 && begin + fresh <= P.n_tokens && has <= P.table_width && len + fresh <= INT32_MAX;
    const int64_t need = fits ? has - had : 0;
    const int64_t off = pages + pg_scan(need, s_sum, &all);
    pages += all;
    const bool ok = fits && (need == 0 || off + need <= count);
    if (live) {
      const int64_t end = begin + fresh;
      const int e = (int)(end < P.n_tokens ? end : P.n_tokens);
      const int2 rec = make_int2((int)len, ok ? (int)(count - 1 - (off < count ? off : count)) : PG_REFUSED);
      if (ALL) {
        s_end[b] = e;
        s_rec[b] = rec;
      } else {
        ((int2*)P.work)[b] = rec;
      }
      P.cu_new[b + 1] = e;
      P.granted[b] = ok;
      P.kv_lens[b] = ok ? (int)(len + fresh) : 0;
      P.lens_out[b] = (int)(ok ? len + fresh : len);
      if (ok && need) taken = (int)(off + need);
    }
  }
  // granted requests that need pages come before the others: the list has lost what the last of them took
  int most = taken;
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const int o = __shfl_xor(most, d);
    most = most > o ? most : o;
  }
  __syncthreads();
  if ((threadIdx.x & (SAH_WAVE - 1)) == 0) s_sum[threadIdx.x / SAH_WAVE] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < PG_NT / SAH_WAVE; ++i) most = most > (int)s_sum[i] ? most : (int)s_sum[i];
    *P.free_count_out = (int)count - most;
    P.cu_new[0] = 0;
  }
  if (ALL) pg_place(P, s_end, s_rec, threadIdx.x, PG_NT);
}

// 12 bytes written per token; a search among the requests' ends, in LDS, for each: 256001 tokens of 1024 requests 4.8 us.
__global__ __launch_bounds__(PG_NT) void k_paged_place(sah_paged_assign_args P) {
  sah_touch_kernargs<sizeof(sah_paged_assign_args)>();
  SAH_DYNAMIC_LDS(s_dyn);
  int2* s_rec = (int2*)s_dyn;
  int* s_end = (int*)(s_rec + P.n_requests);
  for (int b = threadIdx.x; b < P.n_requests; b += PG_NT) {
    s_rec[b] = ((const int2*)P.work)[b];
    s_end[b] = P.cu_new[b + 1];
  }
  __syncthreads();
  pg_place(P, s_end, s_rec, blockIdx.x * PG_NT + threadIdx.x, gridDim.x * PG_NT);
}

// The finished requests' pages, in two kernels of a workgroup a request: how many pages each has, then where the requests before it end in
// the list, and the pages moved behind that, 4 bytes read and 8 written each. An entry below 0 is no page and is not appended. Latency bounds
// both, four dependent reads or writes and three waits in the second: 8 of 64 requests finished, 2048 pages each, 2.6 + 4.6 us; 64 of 1024,
// 500 each, 2.8 + 5.0; 64 of 4096 4.1 + 8.1 (the last one adds up the numbers of all others).
#define PG_BACK_NT 256
#define PG_BACK_E 8   // neighbouring entries a thread
__device__ __forceinline__ int pg_entries(const sah_paged_release_args& P, int b) {  // that a finished request has; 0 of another one
  const int len = P.lens[b], done = P.finished[b];  // (both requested at once)
  const int64_t has = done && len > 0 ? ((int64_t)len + P.page_size - 1) / P.page_size : 0;
  return (int)(has < P.table_width ? has : P.table_width);
}
// a thread's entries of the row from j on
__device__ __forceinline__ void pg_read_entries(const int32_t* row, int j, int has, int (&page)[PG_BACK_E]) {
#pragma unroll
  for (int e = 0; e < PG_BACK_E; ++e) page[e] = j + e < has ? row[j + e] : -1;
}
// work: per request the number of its pages, and beside the first one's that of the list
__global__ __launch_bounds__(PG_BACK_NT) void k_paged_release(sah_paged_release_args P) {
  __shared__ int s_sum[PG_BACK_NT / SAH_WAVE];
  const int b = blockIdx.x, has = pg_entries(P, b);
  const int32_t* row = P.block_table + (int64_t)b * P.table_pitch;
  int n = 0;
  for (int j = (int)threadIdx.x * PG_BACK_E; j < has; j += PG_BACK_NT * PG_BACK_E) {
    int page[PG_BACK_E];
    pg_read_entries(row, j, has, page);
#pragma unroll
    for (int e = 0; e < PG_BACK_E; ++e) n += page[e] >= 0;
  }
  n = sah_wave_sum_i(n);
  if (threadIdx.x % SAH_WAVE == 0) s_sum[threadIdx.x / SAH_WAVE] = n;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < PG_BACK_NT / SAH_WAVE; ++i) n += s_sum[i];
  P.work[2 * b] = n;
  if (b == 0) {
    const int count = *P.free_count;
    P.work[1] = count < 0 ? 0 : (count < P.n_pages ? count : P.n_pages);
  }
}
__global__ __launch_bounds__(PG_BACK_NT) void k_paged_give_back(sah_paged_release_args P) {
  constexpr int NW = PG_BACK_NT / SAH_WAVE;
  __shared__ int64_t s_before[NW];
  __shared__ int s_sum[NW];
  const int b = blockIdx.x, lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  const int has = pg_entries(P, b);
  const bool last = b == P.n_requests - 1;
  if (!has && !last) {
    if (threadIdx.x == 0 && P.finished[b]) P.lens[b] = 0;
    return;
  }
  int32_t* row = P.block_table + (int64_t)b * P.table_pitch;
  int page[PG_BACK_E];
  pg_read_entries(row, (int)threadIdx.x * PG_BACK_E, has, page);  // the first round's, while the sum is taken
  int64_t at = 0;  // where the request's pages begin in the list
  for (int i = threadIdx.x; i < b; i += PG_BACK_NT) at += P.work[2 * i];
  at = (int64_t)sah_lane_u64(sah_wave_incl_scan_u64((uint64_t)at), SAH_WAVE - 1);
  if (lane == 0) s_before[wave] = at;
  __syncthreads();
  at = P.work[1];
  for (int i = 0; i < NW; ++i) at += s_before[i];
  if (threadIdx.x == 0) {
    const int64_t end = at + P.work[2 * b];
    if (last) *P.free_count = (int)(end < P.n_pages ? end : P.n_pages);
    if (P.finished[b]) P.lens[b] = 0;  // (all threads have read it: the wait above)
  }
  for (int j0 = 0; j0 < has; j0 += PG_BACK_NT * PG_BACK_E) {
    const int j = j0 + (int)threadIdx.x * PG_BACK_E;
    if (j0) pg_read_entries(row, j, has, page);
    int n = 0;
#pragma unroll
    for (int e = 0; e < PG_BACK_E; ++e) n += page[e] >= 0;
    const int incl = sah_wave_incl_scan(n);
    __syncthreads();  // the sums of the round before have been read
    if (lane == SAH_WAVE - 1) s_sum[wave] = incl;
    __syncthreads();
    int64_t to = at + incl - n;
    for (int i = 0; i < NW; ++i) {
      to += i < wave ? s_sum[i] : 0;
      at += s_sum[i];
    }
#pragma unroll
    for (int e = 0; e < PG_BACK_E; ++e) {
      if (j + e < has) row[j + e] = -1;
      if (page[e] < 0) continue;
      if (to < P.n_pages) P.free_pages[to] = page[e];  // (a list that is full has no room for more)
      ++to;
    }
  }
}

// A unit is W bytes of a token's keys or values; consecutive threads take consecutive units of a token. Memory: 16384 tokens of 8 heads of
// 128 (bf16, 134 MB moved) 20.6 us, 6.5 TB/s; into a cache that lies in the last-level cache still 13 us, element by element 62. No
// staging, no reuse: nothing is read twice.
template <typename W>
__global__ __launch_bounds__(256) void k_paged_store(sah_paged_store_args P, int units_head, int units_token, int64_t n_units) {
  sah_touch_kernargs<sizeof(sah_paged_store_args) + 16>();
  const int es = P.dtype == SAH_F32 ? 4 : 2;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= n_units) return;
  const int64_t t = u / units_token;
  const int in = (int)(u - t * units_token);
  const int h = in / units_head, c = in - h * units_head;
  const int64_t slot = P.slot_map[t];
  if (slot < 0 || slot >= (int64_t)P.n_pages * P.page_size) return;
  const int64_t page = slot / P.page_size, entry = slot - page * P.page_size;
  const int64_t from_k = (t * P.ks_t + h * P.ks_h) * es, from_v = (t * P.vs_t + h * P.vs_h) * es;
  const W kx = ((const W*)((const char*)P.k + from_k))[c], vx = ((const W*)((const char*)P.v + from_v))[c];
  ((W*)((char*)P.k_cache + (page * P.kcs_p + entry * P.kcs_t + h * P.kcs_h) * es))[c] = kx;
  ((W*)((char*)P.v_cache + (page * P.vcs_p + entry * P.vcs_t + h * P.vcs_h) * es))[c] = vx;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
extern "C" int sah_paged_assign(const sah_paged_assign_args* a) {
  if (!a) return sah_fail(SAH_ENULL, "sah_paged_assign: args is NULL");
  if (a->n_requests <= 0 || a->page_size <= 0 || a->table_width <= 0 || a->n_pages <= 0 || a->n_tokens < 0)
    return sah_fail(SAH_EINVAL, "sah_paged_assign: n_requests, page_size, table_width and n_pages must be > 0, n_tokens >= 0");
  if (a->n_requests > PG_MAX_REQ) return sah_fail(SAH_ESHAPE, "sah_paged_assign: %d requests; at most %d", a->n_requests, PG_MAX_REQ);
  if (a->n_tokens > 1 << 30) return sah_fail(SAH_ESHAPE, "sah_paged_assign: %d tokens; at most 2^30", a->n_tokens);
  if (a->table_pitch < a->table_width) return sah_fail(SAH_EINVAL, "sah_paged_assign: table_pitch is less than table_width");
  if (!a->new_lens || !a->lens || !a->block_table || !a->free_pages || !a->free_count || !a->cu_new || !a->kv_lens || !a->granted ||
      !a->lens_out || !a->free_count_out || !a->work || (a->n_tokens && (!a->slot_map || !a->positions)))
    return sah_fail(SAH_ENULL, "sah_paged_assign: NULL pointer");
  const size_t lds = (size_t)a->n_requests * 12;
  hipStream_t st = (hipStream_t)a->stream;
  if (a->n_tokens <= PG_NT) {
    sah_timed timed("k_paged_assign", a->stream);
    hipLaunchKernelGGL(k_paged_assign<true>, dim3(1), dim3(PG_NT), lds, st, *a);
    return sah_launch_status("sah_paged_assign");
  }
  {
    sah_timed timed("k_paged_assign", a->stream);
    hipLaunchKernelGGL(k_paged_assign<false>, dim3(1), dim3(PG_NT), 0, st, *a);
    if (int rc = sah_launch_status("sah_paged_assign")) return rc;
  }
  sah_timed timed("k_paged_place", a->stream);
  int64_t wgs = ((int64_t)a->n_tokens + PG_NT - 1) / PG_NT;
  hipLaunchKernelGGL(k_paged_place, dim3((unsigned)(wgs < 1024 ? wgs : 1024)), dim3(PG_NT), lds, st, *a);
  return sah_launch_status("sah_paged_assign(place)");
}

extern "C" int sah_paged_release(const sah_paged_release_args* a) {
  if (!a) return sah_fail(SAH_ENULL, "sah_paged_release: args is NULL");
  if (a->n_requests <= 0 || a->page_size <= 0 || a->table_width <= 0 || a->n_pages <= 0)
    return sah_fail(SAH_EINVAL, "sah_paged_release: n_requests, page_size, table_width and n_pages must be > 0");
  if (a->n_requests > PG_MAX_REQ) return sah_fail(SAH_ESHAPE, "sah_paged_release: %d requests; at most %d", a->n_requests, PG_MAX_REQ);
  if (a->table_pitch < a->table_width) return sah_fail(SAH_EINVAL, "sah_paged_release: table_pitch is less than table_width");
  if (!a->finished || !a->lens || !a->block_table || !a->free_pages || !a->free_count || !a->work)
    return sah_fail(SAH_ENULL, "sah_paged_release: NULL pointer");
  hipStream_t st = (hipStream_t)a->stream;
  {
    sah_timed timed("k_paged_release", a->stream);
    hipLaunchKernelGGL(k_paged_release, dim3(a->n_requests), dim3(PG_BACK_NT), 0, st, *a);
    if (int rc = sah_launch_status("sah_paged_release")) return rc;
  }
  sah_timed timed("k_paged_give_back", a->stream);
  hipLaunchKernelGGL(k_paged_give_back, dim3(a->n_requests), dim3(PG_BACK_NT), 0, st, *a);
  return sah_launch_status("sah_paged_release(pages)");
}

extern "C" int sah_paged_store(const sah_paged_store_args* given) {
  if (!given) return sah_fail(SAH_ENULL, "sah_paged_store: args is NULL");
  sah_paged_store_args own = *given;
  const sah_paged_store_args* a = &own;
  // a dimension of one entry has no stride, whatever it is said to be
  if (own.n_tokens == 1) own.ks_t = own.vs_t = 0;
  if (own.Hkv == 1) own.ks_h = own.vs_h = own.kcs_h = own.vcs_h = 0;
  if (own.n_pages == 1) own.kcs_p = own.vcs_p = 0;
  if (own.page_size == 1) own.kcs_t = own.vcs_t = 0;
  if (a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16) return sah_fail(SAH_EDTYPE, "sah_paged_store: dtype %d", a->dtype);
  if (a->n_tokens < 0 || a->Hkv <= 0 || a->D <= 0 || a->n_pages <= 0 || a->page_size <= 0)
    return sah_fail(SAH_EINVAL, "sah_paged_store: Hkv, D, n_pages and page_size must be > 0, n_tokens >= 0");
  if (a->n_tokens == 0) return SAH_OK;
  if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->slot_map) return sah_fail(SAH_ENULL, "sah_paged_store: NULL pointer");
  if (!sah_rows_apart<3>(a->D, {a->kcs_p, a->kcs_t, a->kcs_h}, {a->n_pages, a->page_size, a->Hkv}) ||
      !sah_rows_apart<3>(a->D, {a->vcs_p, a->vcs_t, a->vcs_h}, {a->n_pages, a->page_size, a->Hkv}))
    return sah_fail(SAH_EINVAL, "sah_paged_store: rows of a cache overlap");
  const int es = a->dtype == SAH_F32 ? 4 : 2;
  // 16 bytes at a time where every address allows it, else an element
  const uint64_t all = (uint64_t)a->k | (uint64_t)a->v | (uint64_t)a->k_cache | (uint64_t)a->v_cache |
                       (uint64_t)(es * (a->ks_t | a->ks_h | a->vs_t | a->vs_h | a->kcs_p | a->kcs_t | a->kcs_h | a->vcs_p | a->vcs_t | a->vcs_h | a->D));
  const int wide = all % 16 == 0 ? 16 : es;
  const int64_t units_head = (int64_t)a->D * es / wide, units_token = units_head * a->Hkv, n = units_token * a->n_tokens;
  const int64_t wgs = (n + 255) / 256;
  if (units_token > INT32_MAX || wgs > 0x7fffffff) return sah_fail(SAH_ESHAPE, "sah_paged_store: too many elements");
  hipStream_t st = (hipStream_t)a->stream;
  sah_timed timed("k_paged_store", a->stream);
  if (wide == 16) hipLaunchKernelGGL(k_paged_store<uint4>, dim3((unsigned)wgs), dim3(256), 0, st, *a, (int)units_head, (int)units_token, n);
  else if (wide == 4) hipLaunchKernelGGL(k_paged_store<uint32_t>, dim3((unsigned)wgs), dim3(256), 0, st, *a, (int)units_head, (int)units_token, n);
  else hipLaunchKernelGGL(k_paged_store<uint16_t>, dim3((unsigned)wgs), dim3(256), 0, st, *a, (int)units_head, (int)units_token, n);
  return sah_launch_status("sah_paged_store");
}
