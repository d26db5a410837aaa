// Attention of new tokens over a key-value cache in pages.
#include "sah_common.h"
#include "../../include/sah_serve.h"

#define PA_NT 256
#define PA_NW (PA_NT / SAH_WAVE)
#define PA_MAX_D 256

// A workgroup per row and head; its waves take keys in turn, each with a running maximum and sum of its own, joined in LDS.
template <int DT>
__global__ __launch_bounds__(PA_NT) void k_paged_attn(sah_paged_attention_args P) {
  constexpr int E = PA_MAX_D / SAH_WAVE;
  __shared__ float s_m[PA_NW], s_l[PA_NW], s_acc[PA_NW][PA_MAX_D];
  const int t = blockIdx.x, h = blockIdx.y, hk = h / (P.Hq / P.Hkv);
  const int lane = threadIdx.x & (SAH_WAVE - 1), wave = sah_wave_id();
  int lo = 0, hi = P.n_requests;  // the first request whose rows end behind t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (P.cu_new[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  const int b = lo;
  if (b >= P.n_requests || t < P.cu_new[b]) return;
  int64_t kv = P.kv_lens[b];
  const int64_t most = (int64_t)P.table_width * P.page_size;
  const int64_t p = kv - (P.cu_new[b + 1] - t);
  if (kv > most) kv = most;
  const int64_t end = p + 1 < kv ? p + 1 : kv;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + e * SAH_WAVE;
    q[e] = d < P.D ? sah_load<DT>(P.q, (int64_t)t * P.qs_t + h * P.qs_h + d) * P.scaling : 0.f;
    acc[e] = 0.f;
  }
  for (int64_t j = wave; j < end; j += PA_NW) {
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
    s = sah_wave_sum(s);
    const float m_new = fmaxf(m, s);
    if (m_new == -INFINITY && s == s) continue;  // (a NaN is no maximum, but the row's result)
    const float up = expf(m - m_new), w = expf(s - m_new);
    m = m_new;
    l = l * up + w;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + e * SAH_WAVE;
      if (d < P.D) acc[e] = acc[e] * up + w * sah_load<DT>(P.v, va + d);
    }
  }
  if (lane == 0) { s_m[wave] = m; s_l[wave] = l; }
#pragma unroll
  for (int e = 0; e < E; ++e) s_acc[wave][lane + e * SAH_WAVE] = acc[e];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= P.D) return;
  const float sink = P.sinks ? P.sinks[h] : -INFINITY;
  float M = sink;
  for (int w = 0; w < PA_NW; ++w) M = fmaxf(M, s_m[w]);
  float L = sink == -INFINITY ? 0.f : expf(sink - M), o = 0.f;
  for (int w = 0; w < PA_NW; ++w) {
    const float up = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - M);
    L += s_l[w] * up;
    o += s_acc[w][d] * up;
  }
  sah_store<DT>(P.out, (int64_t)t * P.os_t + h * P.os_h + d, L == 0.f ? 0.f : o / L);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
extern "C" int64_t sah_paged_attention_work_floats(const sah_paged_attention_args* a) { (void)a; return 0; }

extern "C" int sah_paged_attention(const sah_paged_attention_args* a) {
  if (!a) return sah_fail(SAH_ENULL, "sah_paged_attention: args is NULL");
  if (a->dtype != SAH_F32 && a->dtype != SAH_BF16 && a->dtype != SAH_F16) return sah_fail(SAH_EDTYPE, "sah_paged_attention: dtype %d", a->dtype);
  if (a->n_requests <= 0 || a->n_tokens < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->Hq % a->Hkv || a->n_pages <= 0 || a->table_width <= 0 ||
      a->max_context < 0 || a->sink < 0 || a->window < 0)
    return sah_fail(SAH_EINVAL, "sah_paged_attention: bad sizes (n_requests %d, n_tokens %d, heads %d / %d, n_pages %d, table_width %d, max_context %d, "
                    "sink %d, window %d)", a->n_requests, a->n_tokens, a->Hq, a->Hkv, a->n_pages, a->table_width, a->max_context, a->sink, a->window);
  if (a->D <= 0 || a->D % 8 || a->D > PA_MAX_D) return sah_fail(SAH_ESHAPE, "sah_paged_attention: head_dim %d is not a multiple of 8 up to 256", a->D);
  if (a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return sah_fail(SAH_ESHAPE, "sah_paged_attention: page_size %d is not a power of two", a->page_size);
  if ((int64_t)a->table_width * a->page_size > INT32_MAX) return sah_fail(SAH_ESHAPE, "sah_paged_attention: table_width * page_size passes 2^31");
  if (a->table_pitch < a->table_width) return sah_fail(SAH_EINVAL, "sah_paged_attention: table_pitch is less than table_width");
  if (a->n_tokens == 0) return SAH_OK;
  if (!a->q || !a->k || !a->v || !a->block_table || !a->kv_lens || !a->cu_new || !a->out) return sah_fail(SAH_ENULL, "sah_paged_attention: NULL pointer");
  if (a->Hq > 65535) return sah_fail(SAH_ESHAPE, "sah_paged_attention: %d heads", a->Hq);
  const int es = a->dtype == SAH_F32 ? 4 : 2;
  if (((uint64_t)a->q | (uint64_t)a->k | (uint64_t)a->v | (uint64_t)a->out |
       (uint64_t)(es * (a->qs_t | a->qs_h | a->ks_p | a->ks_t | a->ks_h | a->vs_p | a->vs_t | a->vs_h | a->os_t | a->os_h))) % 16)
    return sah_fail(SAH_EINVAL, "sah_paged_attention: addresses and strides must be multiples of 16 bytes");
  if (!(a->scaling == a->scaling)) return sah_fail(SAH_EINVAL, "sah_paged_attention: scaling is NaN");
  hipStream_t st = (hipStream_t)a->stream;
  sah_timed timed("k_paged_attn", a->stream);
  const dim3 grid(a->n_tokens, a->Hq);
  if (a->dtype == SAH_F32) hipLaunchKernelGGL(k_paged_attn<SAH_F32>, grid, dim3(PA_NT), 0, st, *a);
  else if (a->dtype == SAH_BF16) hipLaunchKernelGGL(k_paged_attn<SAH_BF16>, grid, dim3(PA_NT), 0, st, *a);
  else hipLaunchKernelGGL(k_paged_attn<SAH_F16>, grid, dim3(PA_NT), 0, st, *a);
  return sah_launch_status("sah_paged_attention");
}
