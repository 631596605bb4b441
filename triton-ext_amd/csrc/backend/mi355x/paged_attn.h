// Attention of new tokens over a paged cache (tx_cache.h), the plain way: one
// workgroup per token and query head, 256 keys at a time.
#pragma once

#include "rotary.h"

namespace txk {

struct PagedAttnArgs {
  const void *q;
  const uint8_t *kc, *vc;
  const int32_t *table, *kv_len, *cu_q;
  const float *k_scale, *v_scale;
  void *o;
  float *lse;
  uint32_t *counters;
  uint8_t *parts;
  int64_t T, pages, table_width, table_s;
  int64_t q_st, q_sh, o_st, o_sh, k_sp, k_st, k_sh, v_sp, v_st, v_sh;
  int32_t B, Hq, Hkv, head_dim, page_shift, causal, window;
  float qk_scale; // sm_scale / ln 2
};

__device__ __forceinline__ float e4m3_to_f32(uint8_t x) {
  return __builtin_amdgcn_cvt_f32_fp8(x, 0);
}
template <class T, class C> __device__ __forceinline__ float cache_f32(const uint8_t *row, int d) {
  if constexpr (std::is_same<C, uint8_t>::value)
    return e4m3_to_f32(row[d]);
  else
    return elt_to_f32(reinterpret_cast<const T *>(row)[d]);
}

template <class T, class C>
__global__ void __launch_bounds__(256) paged_attn_plain_kernel(PagedAttnArgs p) {
  __shared__ float qs[256], ps[256], red[4];
  __shared__ int64_t pg[256];
  const int tid = threadIdx.x, h = blockIdx.y, hk = h / (p.Hq / p.Hkv);
  const int64_t t = blockIdx.x;
  int b = (int)t;
  int64_t pos, len = 0;
  if (p.cu_q) {
    b = sequence_of(p.cu_q, p.B, t);
    const int64_t first = p.cu_q[b], last = p.cu_q[b + 1];
    pos = (int64_t)p.kv_len[b] - last + t;
    if (t >= first && t < last)
      len = p.kv_len[b];
  } else {
    pos = (int64_t)p.kv_len[b] - 1;
    len = p.kv_len[b];
  }
  int64_t lo = p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
  int64_t hi = p.causal && pos + 1 < len ? pos + 1 : len;
  const int64_t most = p.table_width << p.page_shift;
  hi = hi < most ? hi : most;
  if (tid < p.head_dim)
    qs[tid] = elt_to_f32(static_cast<const T *>(p.q)[t * p.q_st + h * p.q_sh + tid]) *
              (p.k_scale ? p.k_scale[hk] : 1.f);
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int64_t j0 = lo; j0 < hi; j0 += 256) {
    __syncthreads();
    const int64_t j = j0 + tid;
    int64_t page = -1;
    if (j < hi)
      page = p.table[b * p.table_s + (j >> p.page_shift)];
    if (page >= p.pages)
      page = -1;
    float s = -INFINITY;
    const int64_t slot = j & ((1 << p.page_shift) - 1);
    if (page >= 0) {
      const uint8_t *row = p.kc + (page * p.k_sp + slot * p.k_st + hk * p.k_sh) * sizeof(C);
      s = 0.f;
      for (int d = 0; d < p.head_dim; ++d)
        s += qs[d] * cache_f32<T, C>(row, d);
      s *= p.qk_scale;
    }
    float mx = s;
    for (int d = 32; d; d /= 2)
      mx = fmaxf(mx, __shfl_xor(mx, d));
    if ((tid & 63) == 0)
      red[tid >> 6] = mx;
    __syncthreads();
    const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float base = mn == -INFINITY ? 0.f : mn;
    ps[tid] = exp2f(s - base);
    pg[tid] = page < 0 ? -1 : page * p.v_sp + slot * p.v_st + hk * p.v_sh;
    __syncthreads();
    const float alpha = exp2f(m - base);
    l *= alpha;
    acc *= alpha;
    m = mn;
    const int n = hi - j0 < 256 ? (int)(hi - j0) : 256;
    for (int i = 0; i < n; ++i) {
      if (pg[i] < 0)
        continue;
      l += ps[i];
      if (tid < p.head_dim)
        acc += ps[i] * cache_f32<T, C>(p.vc + pg[i] * sizeof(C), tid);
    }
  }
  if (tid < p.head_dim)
    static_cast<T *>(p.o)[t * p.o_st + h * p.o_sh + tid] =
        (T)(l > 0.f ? acc / l * (p.v_scale ? p.v_scale[hk] : 1.f) : 0.f);
  if (tid == 0 && p.lse)
    p.lse[t * p.Hq + h] = l > 0.f ? m + log2f(l) : -INFINITY;
}

} // namespace txk
