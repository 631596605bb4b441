// New tokens into a 4-bit paged cache, and tokens out of any paged cache (tx_cache4.h).
//
// Append: a lane takes 8 adjacent dims of a head, so that a block's lanes (4, or 2 under e4m3
// scales) are neighbours that find its largest magnitude by two DPP moves.  Rotated dims need
// their partners, rot_dim / 2 further (halves) or in the same 8 (interleaved): the lane reads
// them too.  A thread forms its 8 (or 4) sines once and goes through the token's heads, every
// head_lanes-th of them.
//
// Read: the same threads; a lane turns 8 dims into 16 or 32 bytes.  Both are bound by memory.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "cache4.h"
#include "rotary.h"

namespace txk {

struct BlockScales { // bytes from one (page, token, head, block) to the next
  uint8_t *s;
  int64_t sp, st, sh, sb;
};

struct Append4Args {
  AppendArgs a; // (strides of the caches in bytes)
  BlockScales ks, vs;
  int32_t lo, hi; // exponents of MX32
};

// Token t of the call: its sequence, its position, its page (-1: none) and whether it is of a
// sequence at all.
struct TokenPlace {
  int b;
  int64_t pos, page;
  bool mine;
};
__device__ __forceinline__ TokenPlace token_place(int64_t t, const int32_t *cu_q, const int32_t *kv_len,
                                                  int B, const int32_t *table, int64_t table_s,
                                                  int64_t table_width, int64_t pages, int page_shift) {
  TokenPlace r;
  r.b = (int)t, r.page = -1, r.mine = true;
  if (cu_q) {
    r.b = sequence_of(cu_q, B, t);
    const int64_t first = cu_q[r.b], last = cu_q[r.b + 1];
    r.mine = t >= first && t < last;
    r.pos = kv_len[r.b] - last + t;
  } else {
    r.pos = (int64_t)kv_len[r.b] - 1;
  }
  const int64_t e = r.pos >> page_shift;
  if (r.mine && r.pos >= 0 && e < table_width) {
    r.page = table[r.b * table_s + e];
    if (r.page >= pages)
      r.page = -1;
  }
  return r;
}

// 8 elements from p on; WHOLE: in one access.
template <class T, bool WHOLE>
__device__ __forceinline__ void load8(const T *p, EltVec<T, 8> &x) {
  if constexpr (WHOLE) {
    x = *reinterpret_cast<const EltVec<T, 8> *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x.v[i] = p[i];
  }
}
template <class T, bool WHOLE>
__device__ __forceinline__ void store8(T *p, const float (&y)[8]) {
  EltVec<T, 8> r;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    r.v[i] = (T)y[i];
  if constexpr (!WHOLE) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      p[i] = r.v[i];
  } else if constexpr (sizeof(T) == 4) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    reinterpret_cast<f4 *>(p)[0] = f4{y[0], y[1], y[2], y[3]};
    reinterpret_cast<f4 *>(p)[1] = f4{y[4], y[5], y[6], y[7]};
  } else {
    *reinterpret_cast<EltVec<T, 8> *>(p) = r;
  }
}

// The turn of 8 adjacent dims: y = x c + partner s (with the sign of each dim's half).
template <bool INTER> struct Turn8 {
  bool any; // of the 8 dims is rotated
  int dim, rot;
  float c[INTER ? 4 : 8], s[INTER ? 4 : 8];

  __device__ __forceinline__ Turn8(int item, int rot_dim, double pos, const float *inv_freq, float scale)
      : any(8 * item < rot_dim), dim(8 * item), rot(rot_dim) {
    if (!any)
      return;
#pragma unroll
    for (int i = 0; i < (INTER ? 4 : 8); ++i) {
      const int d = INTER ? dim + 2 * i : dim + i;
      c[i] = 1.f, s[i] = 0.f;
      if (d < rot) {
        const bool second = !INTER && d >= rot / 2;
        turn_of(pos, inv_freq[INTER ? d / 2 : second ? d - rot / 2 : d], scale, !INTER && !second, c[i], s[i]);
      }
    }
  }
  // The partners of the 8 dims (halves; a dim past rot: itself).
  template <class T, bool WHOLE>
  __device__ __forceinline__ void load_partners(const T *head, EltVec<T, 8> &x) const {
    if constexpr (!INTER) {
      if constexpr (WHOLE) { // (rot / 2 is a multiple of 8)
        load8<T, true>(head + (any ? dim < rot / 2 ? dim + rot / 2 : dim - rot / 2 : dim), x);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = dim + i;
          x.v[i] = head[d >= rot ? d : d < rot / 2 ? d + rot / 2 : d - rot / 2];
        }
      }
    }
  }
  template <class T>
  __device__ __forceinline__ void apply(const EltVec<T, 8> &x, const EltVec<T, 8> &partner, bool turn,
                                        float (&y)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = elt_to_f32(x.v[i]);
    if (!any || !turn)
      return;
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = y[2 * i], b = y[2 * i + 1];
        if (dim + 2 * i < rot) {
          y[2 * i] = a * c[i] - b * s[i];
          y[2 * i + 1] = b * c[i] + a * s[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (dim + i < rot)
          y[i] = y[i] * c[i] + elt_to_f32(partner.v[i]) * s[i];
    }
  }
};

// Heads in the order q, k, v.
template <class T, bool NV, bool INTER, bool WHOLE>
__global__ void __launch_bounds__(256) paged_append4_kernel(Append4Args args) {
  const AppendArgs &p = args.a;
  const RotaryPlace at(p.token_threads, p.items, false);
  const int64_t t = at.tok;
  if (t >= p.T)
    return;
  const TokenPlace pl = token_place(t, p.cu_q, p.kv_len, p.B, p.table, p.table_s, p.table_width, p.pages,
                                    p.page_shift);
  const int64_t slot = pl.pos & ((1 << p.page_shift) - 1);
  const Turn8<INTER> turn(at.item, p.rot, (double)pl.pos, p.inv_freq, p.scale);
  constexpr int LANES = NV ? 2 : 4; // of a block
  // (a token without a page: its q alone)
  const int heads = pl.page < 0 ? p.Hq : p.Hq + 2 * p.Hkv;
  for (int h0 = at.lane; h0 < heads; h0 += kHeadBatch * p.head_lanes) {
    EltVec<T, 8> x[kHeadBatch], partner[kHeadBatch];
#pragma unroll
    for (int k = 0; k < kHeadBatch; ++k) {
      const int hh = h0 + k * p.head_lanes, h = hh < heads ? hh : h0;
      const bool is_q = h < p.Hq, is_k = h < p.Hq + p.Hkv;
      const int hk = h - p.Hq - (is_k ? 0 : p.Hkv);
      const T *src = is_q   ? static_cast<const T *>(p.q) + t * p.q_st + h * p.q_sh
                     : is_k ? static_cast<const T *>(p.k) + t * p.k_st + hk * p.k_sh
                            : static_cast<const T *>(p.v) + t * p.v_st + hk * p.v_sh;
      load8<T, WHOLE>(src + turn.dim, x[k]);
      if (is_k)
        turn.template load_partners<T, WHOLE>(src, partner[k]);
    }
#pragma unroll
    for (int k = 0; k < kHeadBatch; ++k) {
      const int h = h0 + k * p.head_lanes;
      if (h >= heads)
        break;
      float y[8];
      if (h < p.Hq) {
        turn.template apply<T>(x[k], partner[k], pl.mine, y);
        store8<T, WHOLE>(static_cast<T *>(p.q_out) + t * p.o_st + h * p.o_sh + turn.dim, y);
        continue;
      }
      const bool is_k = h < p.Hq + p.Hkv;
      const int hk = h - p.Hq - (is_k ? 0 : p.Hkv);
      turn.template apply<T>(x[k], partner[k], is_k, y);
      const float *sc = is_k ? p.k_scale : p.v_scale;
      if (sc) {
        const float f = sc[hk];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          y[i] = y[i] / f;
      }
      const uint32_t scale = block4_scale<NV>(block4_max<LANES>(y), args.lo, args.hi);
      uint8_t *dst = is_k ? p.kc + pl.page * p.kc_sp + slot * p.kc_st + hk * p.kc_sh
                          : p.vc + pl.page * p.vc_sp + slot * p.vc_st + hk * p.vc_sh;
      *reinterpret_cast<uint32_t *>(dst + 4 * at.item) = block4_codes<NV>(y, scale);
      if (at.item % LANES == 0) {
        const int64_t blk = at.item / LANES;
        if (is_k)
          args.ks.s[pl.page * args.ks.sp + slot * args.ks.st + hk * args.ks.sh + blk * args.ks.sb] = scale;
        else
          args.vs.s[pl.page * args.vs.sp + slot * args.vs.st + hk * args.vs.sh + blk * args.vs.sb] = scale;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Tokens out of a cache
// ---------------------------------------------------------------------------

struct ReadArgs {
  const uint8_t *kc, *vc;
  BlockScales ks, vs;
  const int32_t *table, *kv_len, *cu_q;
  const float *k_scale, *v_scale;
  void *k, *v;
  int64_t T, pages, table_width, table_s;
  int64_t kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh; // bytes
  int64_t k_st, k_sh, v_st, v_sh;                   // elements
  int32_t B, Hkv, head_dim, items, head_lanes, page_shift, token_threads;
};

struct E4m3 {};              // caches of bytes
template <bool NV> struct E2m1 {};
template <class C> struct IsE2m1 : std::false_type {};
template <bool NV> struct IsE2m1<E2m1<NV>> : std::true_type {
  static constexpr bool nv = NV;
};

// VEC dims from dim d on of a head, as loaded.
template <class C, int VEC> struct ReadItem {
  static constexpr int BYTES = VEC * (std::is_same<C, E4m3>::value ? 1 : 2);
  EltVec<uint8_t, BYTES> x;
  __device__ __forceinline__ void load(const uint8_t *head, int d, const BlockScales &, const uint8_t *) {
    x = *reinterpret_cast<const EltVec<uint8_t, BYTES> *>(head + d * (BYTES / VEC));
  }
  __device__ __forceinline__ void values(float (&y)[VEC]) const {
    if constexpr (std::is_same<C, E4m3>::value) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        y[i] = __builtin_amdgcn_cvt_f32_fp8(x.v[i], 0);
    } else {
      const EltVec<C, VEC> e = __builtin_bit_cast(EltVec<C, VEC>, x);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        y[i] = elt_to_f32(e.v[i]);
    }
  }
};
template <bool NV> struct ReadItem<E2m1<NV>, 8> {
  uint32_t w, s;
  __device__ __forceinline__ void load(const uint8_t *head, int d, const BlockScales &bs, const uint8_t *scales) {
    w = *reinterpret_cast<const uint32_t *>(head + d / 2);
    s = scales[(d / (NV ? 16 : 32)) * bs.sb];
  }
  __device__ __forceinline__ void values(float (&y)[8]) const { codes4_f32<NV>(w, s, y); }
};

// Heads in the order k, v.
template <class C, class O, int VEC, bool WHOLE>
__global__ void __launch_bounds__(256) paged_read_kernel(ReadArgs p) {
  const RotaryPlace at(p.token_threads, p.items, false);
  const int64_t t = at.tok;
  if (t >= p.T)
    return;
  const TokenPlace pl = token_place(t, p.cu_q, p.kv_len, p.B, p.table, p.table_s, p.table_width, p.pages,
                                    p.page_shift);
  const int64_t slot = pl.pos & ((1 << p.page_shift) - 1);
  const int d = at.item * VEC;
  const int heads = 2 * p.Hkv;
  for (int h0 = at.lane; h0 < heads; h0 += kHeadBatch * p.head_lanes) {
    ReadItem<C, VEC> x[kHeadBatch];
    if (pl.page >= 0) {
#pragma unroll
      for (int k = 0; k < kHeadBatch; ++k) {
        const int hh = h0 + k * p.head_lanes, h = hh < heads ? hh : h0;
        const bool is_k = h < p.Hkv;
        const int hk = is_k ? h : h - p.Hkv;
        const uint8_t *src = is_k ? p.kc + pl.page * p.kc_sp + slot * p.kc_st + hk * p.kc_sh
                                  : p.vc + pl.page * p.vc_sp + slot * p.vc_st + hk * p.vc_sh;
        const BlockScales &bs = is_k ? p.ks : p.vs;
        x[k].load(src, d, bs, bs.s + pl.page * bs.sp + slot * bs.st + hk * bs.sh);
      }
    }
#pragma unroll
    for (int k = 0; k < kHeadBatch; ++k) {
      const int h = h0 + k * p.head_lanes;
      if (h >= heads)
        break;
      const bool is_k = h < p.Hkv;
      const int hk = is_k ? h : h - p.Hkv;
      float y[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        y[i] = 0.f;
      if (pl.page >= 0) {
        x[k].values(y);
        if (const float *sc = is_k ? p.k_scale : p.v_scale) {
          const float f = sc[hk];
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            y[i] *= f;
        }
      }
      O *out = is_k ? static_cast<O *>(p.k) + t * p.k_st + hk * p.k_sh
                    : static_cast<O *>(p.v) + t * p.v_st + hk * p.v_sh;
      if constexpr (VEC == 8)
        store8<O, WHOLE>(out + d, y);
      else
        out[d] = (O)y[0];
    }
  }
}

} // namespace txk
