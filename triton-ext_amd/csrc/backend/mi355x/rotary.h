// Rotary positions, and new tokens written into a paged cache.
//
// A pair (x1, x2) at position p with frequency f goes to (x1 c - x2 s, x2 c + x1 s),
// c + i s = scale e^(i p f).  The angle's turn is taken in 64 bits (at a position of
// 10^6 the product in fp32 is off by 0.06), sine and cosine of the reduced turn and
// the rotation in fp32, and the result is rounded once.
//
// Every thread takes the same piece of a token's heads: `item` of one head is VEC
// elements of each half of the rotated part (halves layout), VEC adjacent elements
// (interleaved), or VEC elements past rot_dim, which are copied.  So it forms its
// VEC (or VEC / 2) sines once and goes through the token's heads, every
// head_lanes-th of them, kHeadBatch at a time: their 16-byte loads are all under way before
// the first store.  Bound by memory: (4, 32, 4096, 64) in fp16 with 32 dims rotated 23.9 us, 5.6
// TB/s (one head at a time 32.9); 9001 tokens of 32 + 2 x 8 heads of 128 into an e4m3 cache 40.9 us, 5.0
// TB/s (58.6).  Loads are non-temporal: what a projection left is read once (25.8 and 46.7 without).
// A step's few tokens take 3.5 .. 4.5 us, less than the call on the host.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "tile_common.h"

namespace txk {

struct RotaryArgs {
  const void *x;
  const void *pos;
  const float *inv_freq;
  void *out;
  int64_t N, tokens; // tokens: Z * N
  int32_t token_threads, token_fast; // RotaryPlace
  int64_t pos_sz, x_sz, x_sn, x_sh, o_sz, o_sn, o_sh;
  int32_t H, head_dim, rot, items, head_lanes, pos64, inverse;
  float scale;
};

struct AppendArgs {
  const void *q, *k, *v;
  void *q_out;
  uint8_t *kc, *vc;
  const int32_t *table, *kv_len, *cu_q;
  const float *inv_freq, *k_scale, *v_scale;
  int64_t T, pages, table_width, table_s;
  int64_t q_st, q_sh, o_st, o_sh, k_st, k_sh, v_st, v_sh;
  int64_t kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh;
  int32_t B, Hq, Hkv, head_dim, rot, items, head_lanes, page_shift;
  int32_t token_threads;
  float scale;
};

constexpr int kHeadBatch = 4; // heads that a thread has under way

// What a thread does: `item` of heads lane, lane + head_lanes, .. of a token.  A token has
// token_threads = items x head_lanes threads, items fastest; a workgroup of 256 has whole tokens, or
// a token whole workgroups.  token_fast (heads further apart than tokens): token_threads =
// items, and the lane is blockIdx.y.
struct RotaryPlace {
  int64_t tok;
  int item, lane;
  __device__ __forceinline__ RotaryPlace(uint32_t token_threads, uint32_t items, bool token_fast) {
    uint32_t in;
    if (token_threads <= 256) {
      const uint32_t per = 256 / token_threads, t = threadIdx.x / token_threads;
      tok = t < per ? (int64_t)blockIdx.x * per + t : INT64_MAX;
      in = threadIdx.x - t * token_threads;
    } else {
      const uint32_t blocks = (token_threads + 255) / 256, t = blockIdx.x / blocks;
      in = (blockIdx.x - t * blocks) * 256 + threadIdx.x;
      tok = in < token_threads ? (int64_t)t : INT64_MAX;
    }
    const uint32_t l = in / items;
    item = in - l * items;
    lane = token_fast ? blockIdx.y : l;
  }
};

__device__ __forceinline__ float elt_to_f32(float x) { return x; }
__device__ __forceinline__ float elt_to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float elt_to_f32(__bf16 x) { return (float)x; }

template <class T, int VEC> struct alignas(sizeof(T) * VEC) EltVec {
  T v[VEC];
};
template <class T, int VEC>
__device__ __forceinline__ void store_f32(T *p, const float (&f)[VEC]) {
  EltVec<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    r.v[i] = (T)f[i];
  *reinterpret_cast<EltVec<T, VEC> *>(p) = r;
}

// cos and sin of position * f, times scale.
__device__ __forceinline__ void turn_of(double pos, float f, float scale, bool inverse, float &c,
                                        float &s) {
  double t = pos * (double)f * 0.15915494309189535; // turns
  t -= rint(t);
  float si, co;
  sincospif(2.0f * (float)t, &si, &co);
  c = co * scale;
  s = (inverse ? -si : si) * scale;
}

// What one item of a head is: offsets of its one or two runs of VEC elements, and
// the sines of its pairs.
template <int VEC, bool INTER> struct RotaryItem {
  static constexpr int P = INTER ? (VEC > 1 ? VEC / 2 : 1) : VEC;
  int at, second; // second < 0: one run; interleaved VEC 1: the pair's other element
  bool rotate;
  float c[P], s[P];

  __device__ __forceinline__ RotaryItem(int item, int rot, double pos, const float *inv_freq,
                                        float scale, bool inverse) {
    // pair items come first
    const int step = INTER ? (VEC > 1 ? VEC : 2) : VEC;
    const int pairs = INTER ? rot / step : rot / 2 / VEC;
    rotate = item < pairs;
    if (rotate) {
      at = item * step;
      second = INTER ? (VEC > 1 ? -1 : at + 1) : at + rot / 2;
#pragma unroll
      for (int i = 0; i < P; ++i)
        turn_of(pos, inv_freq[INTER ? at / 2 + i : at + i], scale, inverse, c[i], s[i]);
    } else {
      at = rot + (item - pairs) * VEC;
      second = -1;
#pragma unroll
      for (int i = 0; i < P; ++i)
        c[i] = 1.f, s[i] = 0.f;
    }
  }
  // The item of one head, and rotated (or not): y1 goes to `at`, y2 to `second`.
  template <class T>
  __device__ __forceinline__ void load(const T *head, EltVec<T, VEC> &x1, EltVec<T, VEC> &x2) const {
    if constexpr (sizeof(T) * VEC == 16) {
      typedef uint32_t q4 __attribute__((ext_vector_type(4)));
      const T *const head2 = head + (second >= 0 ? second : at);
      x1 = __builtin_bit_cast(EltVec<T, VEC>,
                              __builtin_nontemporal_load(reinterpret_cast<const q4 *>(head + at)));
      x2 = __builtin_bit_cast(EltVec<T, VEC>,
                              __builtin_nontemporal_load(reinterpret_cast<const q4 *>(head2)));
    } else {
      x1 = *reinterpret_cast<const EltVec<T, VEC> *>(head + at);
      x2 = *reinterpret_cast<const EltVec<T, VEC> *>(head + (second >= 0 ? second : at));
    }
  }
  template <class T>
  __device__ __forceinline__ void apply(const EltVec<T, VEC> &x1, const EltVec<T, VEC> &x2,
                                        bool rot_it, float (&y1)[VEC], float (&y2)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      y1[i] = elt_to_f32(x1.v[i]), y2[i] = elt_to_f32(x2.v[i]);
    if (!rotate || !rot_it)
      return;
    if constexpr (INTER && VEC > 1) {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const float a = y1[2 * i], b = y1[2 * i + 1];
        y1[2 * i] = a * c[i] - b * s[i];
        y1[2 * i + 1] = b * c[i] + a * s[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float a = y1[i], b = y2[i];
        y1[i] = a * c[i] - b * s[i];
        y2[i] = b * c[i] + a * s[i];
      }
    }
  }
};

template <class T, int VEC, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs p) {
  const RotaryPlace at(p.token_threads, p.items, p.token_fast);
  const int64_t tok = at.tok;
  if (tok >= p.tokens)
    return;
  const int64_t z = p.tokens == p.N ? 0 : tok / p.N, n = tok - z * p.N;
  const int64_t pi = z * p.pos_sz + n;
  const double pos = p.pos64 ? (double)static_cast<const int64_t *>(p.pos)[pi]
                             : (double)static_cast<const int32_t *>(p.pos)[pi];
  const RotaryItem<VEC, INTER> it(at.item, p.rot, pos, p.inv_freq, p.scale, p.inverse);
  const T *x = static_cast<const T *>(p.x) + z * p.x_sz + n * p.x_sn;
  T *o = static_cast<T *>(p.out) + z * p.o_sz + n * p.o_sn;
  for (int h0 = at.lane; h0 < p.H; h0 += kHeadBatch * p.head_lanes) {
    EltVec<T, VEC> x1[kHeadBatch], x2[kHeadBatch];
#pragma unroll
    for (int k = 0; k < kHeadBatch; ++k) {
      const int h = h0 + k * p.head_lanes;
      it.template load<T>(x + (h < p.H ? h : h0) * p.x_sh, x1[k], x2[k]);
    }
#pragma unroll
    for (int k = 0; k < kHeadBatch; ++k) {
      const int h = h0 + k * p.head_lanes;
      if (h >= p.H)
        break;
      float y1[VEC], y2[VEC];
      it.template apply<T>(x1[k], x2[k], true, y1, y2);
      T *oh = o + h * p.o_sh;
      store_f32<T, VEC>(oh + it.at, y1);
      if (it.second >= 0)
        store_f32<T, VEC>(oh + it.second, y2);
    }
  }
}

// The sequence of token t: the largest b with cu_q[b] <= t (cu_q ascends).
__device__ __forceinline__ int sequence_of(const int32_t *cu_q, int B, int64_t t) {
  int lo = 0, hi = B; // cu_q[lo] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu_q[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint8_t f32_to_e4m3(float x) {
  // saturates at 448 (the conversion itself makes NaN past it); NaN stays NaN
  x = x > 448.f ? 448.f : x < -448.f ? -448.f : x;
  return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xff);
}

template <class T, class C, int VEC>
__device__ __forceinline__ void store_cache(uint8_t *head, int at, const float (&y)[VEC],
                                            float scale) {
  if constexpr (std::is_same<C, uint8_t>::value) {
    EltVec<uint8_t, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      r.v[i] = f32_to_e4m3(y[i] / scale);
    *reinterpret_cast<EltVec<uint8_t, VEC> *>(head + at) = r;
  } else {
    store_f32<T, VEC>(reinterpret_cast<T *>(head) + at, y);
  }
}

// C: T, or uint8_t for e4m3.  Heads in the order q, k, v.
template <class T, class C, int VEC, bool INTER>
__global__ void __launch_bounds__(256) paged_append_kernel(AppendArgs p) {
  const RotaryPlace at(p.token_threads, p.items, false);
  const int64_t t = at.tok;
  if (t >= p.T)
    return;
  // Token t's sequence b, position and place in the cache (page < 0: none).
  int b = (int)t;
  int64_t pos = -1, page = -1;
  bool mine = true;
  if (p.cu_q) {
    b = sequence_of(p.cu_q, p.B, t);
    const int64_t first = p.cu_q[b], last = p.cu_q[b + 1];
    mine = t >= first && t < last;
    pos = p.kv_len[b] - last + t;
  } else {
    pos = (int64_t)p.kv_len[b] - 1;
  }
  const int64_t e = pos >> p.page_shift;
  if (mine && pos >= 0 && e < p.table_width) {
    page = p.table[b * p.table_s + e];
    if (page >= p.pages)
      page = -1;
  }
  const int64_t slot = pos & ((1 << p.page_shift) - 1);
  const RotaryItem<VEC, INTER> it(at.item, p.rot, (double)pos, p.inv_freq, p.scale, false);
  // (a token without a page: its q alone)
  const int heads = page < 0 ? p.Hq : p.Hq + 2 * p.Hkv;
  for (int h0 = at.lane; h0 < heads; h0 += kHeadBatch * p.head_lanes) {
    EltVec<T, VEC> x1[kHeadBatch], x2[kHeadBatch];
#pragma unroll
    for (int k = 0; k < kHeadBatch; ++k) {
      const int hh = h0 + k * p.head_lanes, h = hh < heads ? hh : h0;
      const bool is_q = h < p.Hq, is_k = h < p.Hq + p.Hkv;
      const int hk = h - p.Hq - (is_k ? 0 : p.Hkv);
      const T *src = is_q   ? static_cast<const T *>(p.q) + t * p.q_st + h * p.q_sh
                     : is_k ? static_cast<const T *>(p.k) + t * p.k_st + hk * p.k_sh
                            : static_cast<const T *>(p.v) + t * p.v_st + hk * p.v_sh;
      it.template load<T>(src, x1[k], x2[k]);
    }
#pragma unroll
    for (int k = 0; k < kHeadBatch; ++k) {
      const int h = h0 + k * p.head_lanes;
      if (h >= heads)
        break;
      float y1[VEC], y2[VEC];
      if (h < p.Hq) {
        it.template apply<T>(x1[k], x2[k], mine, y1, y2);
        T *o = static_cast<T *>(p.q_out) + t * p.o_st + h * p.o_sh;
        store_f32<T, VEC>(o + it.at, y1);
        if (it.second >= 0)
          store_f32<T, VEC>(o + it.second, y2);
        continue;
      }
      const bool is_k = h < p.Hq + p.Hkv;
      const int hk = h - p.Hq - (is_k ? 0 : p.Hkv);
      it.template apply<T>(x1[k], x2[k], is_k, y1, y2);
      const float *sc = is_k ? p.k_scale : p.v_scale;
      const float scale = sc ? sc[hk] : 1.f;
      uint8_t *dst = is_k ? p.kc + (page * p.kc_sp + slot * p.kc_st + hk * p.kc_sh) * sizeof(C)
                          : p.vc + (page * p.vc_sp + slot * p.vc_st + hk * p.vc_sh) * sizeof(C);
      store_cache<T, C, VEC>(dst, it.at, y1, scale);
      if (it.second >= 0)
        store_cache<T, C, VEC>(dst, it.second, y2, scale);
    }
  }
}

} // namespace txk
