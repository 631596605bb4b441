// New tokens into a 4-bit paged cache, and tokens out of any paged cache (tx_cache4.h).
//
// Append: a lane takes 8 adjacent dims of a head, or 8 of each half of its rotated dims, so that a
// block's lanes (4, or 2 under e4m3 scales) are neighbours that find its largest magnitude by two DPP
// moves.  A token's sines are formed once, a pair a thread, and go through LDS; a thread then goes
// through the token's heads, every head_lanes-th of them.
//
// Read: the same threads; a lane turns 8 dims into 16 or 32 bytes.
//
// Both are bound by memory.  Append, 9001 tokens of 32 + 2 * 8 heads of 128 in bf16, e4m3 scales: 44 us,
// 4.5 TB/s (a copy reaches 5.07); 48 tokens: 5 us, the latency of the table, the sines and the values one
// after the other.  With a thread for 8 dims of one head, its sines its own, that prompt and its reading back
// took 90 us, now 56.  Read, 156000 tokens of 2 * 8 heads of 128 into bf16: 167 us, 5.0 TB/s (so: 233).
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "cache4.h"
#include "rotary.h"
#include "sine_share.h"

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

// 8 elements from p on; WHOLE: in one access; NT: data that is read once.
template <class T, bool WHOLE, bool NT>
__device__ __forceinline__ void load8(const T *p, EltVec<T, 8> &x) {
  if constexpr (WHOLE && NT) {
    typedef uint32_t w4 __attribute__((ext_vector_type(4)));
    x = __builtin_bit_cast(EltVec<T, 8>, __builtin_nontemporal_load(reinterpret_cast<const w4 *>(p)));
  } else if constexpr (WHOLE) {
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

// cos and sin of position * f, times scale, in 64 bits and rounded once: a key is quantised after its
// rotation, and one that lies at a border of two codes goes to either by the last bit of its sines.  (The
// second constant is what the first leaves of 1 / 2 pi: the turn is off by less than 2^-53 then.)
__device__ __forceinline__ float2_t turn4_of(double pos, float f, float scale) {
  const double a = pos * (double)f, n = rint(a * 0.15915494309189535);
  const double turn = fma(a, -9.839338337591243e-18, fma(a, 0.15915494309189535, -n));
  double s, c;
  sincospi(2.0 * turn, &s, &c);
  return float2_t{(float)(c * scale), (float)(s * scale)};
}
// A rotated dim, x c + z s with its partner z: both products and their sum rounded to fp32 (not
// contracted, so that both dims of a pair, of every form, are rounded alike).
__device__ __forceinline__ float turned4(float x, float c, float z, float s) {
#pragma clang fp contract(off)
  return x * c + z * s;
}

// How a thread has the dims of a head: 8 adjacent ones whose partners are elsewhere (any rot_dim), 8 of
// each half of the rotated dims and of those past them (blocks lie within a half), or 8 of interleaved pairs.
enum { kRunAlone = 0, kRunHalves = 1, kRunPairs = 2 };
constexpr int kAppendSines = 2048; // pairs of a workgroup's tokens in LDS

template <class T, bool NV, int MODE, bool WHOLE>
__global__ void __launch_bounds__(256) paged_append4_kernel(Append4Args args) {
  constexpr int RUNS = MODE == kRunHalves ? 2 : 1, LANES = NV ? 2 : 4; // LANES of a block
  constexpr int BATCH = RUNS == 2 ? 2 : 4;                             // heads that a thread has under way
  __shared__ float2_t sines[kAppendSines];
  const AppendArgs &p = args.a;
  const RotaryPlace at(p.token_threads, p.items, false);
  const int64_t t = at.tok;
  const bool on = t < p.T;
  TokenPlace pl = {};
  if (on)
    pl = token_place(t, p.cu_q, p.kv_len, p.B, p.table, p.table_s, p.table_width, p.pages, p.page_shift);
  const int rot = p.rot, half = rot / 2;

  // The token's sines, a pair a thread, in LDS; heads of more pairs than that: each thread its own.
  const SineShare mine = sine_share(threadIdx.x, p.token_threads, at.lane * p.items + at.item);
  const int mine0 = (int)mine.token * half;
  const bool shared = (p.token_threads <= 256 ? 256 / p.token_threads : 1) * half <= kAppendSines;
  if (shared && on)
    for (int i = mine.first; i < half; i += mine.step)
      sines[mine0 + i] = turn4_of((double)pl.pos, p.inv_freq[i], p.scale);
  __syncthreads();
  if (!on)
    return;

  // dims d[r] .. d[r] + 7
  int d[RUNS];
  if constexpr (MODE == kRunHalves) {
    const int pairs = rot / 16, i = at.item < pairs ? at.item : at.item - pairs;
    const int from = at.item < pairs ? 0 : rot, n = at.item < pairs ? rot : p.head_dim - rot;
    d[0] = from + 8 * i, d[RUNS - 1] = from + n / 2 + 8 * i;
  } else {
    d[0] = 8 * at.item;
  }
  const bool turned = d[0] < rot;
  // of pair (dims j and j + half; or 2 j and 2 j + 1) that dim d[0] + i (or 2 i) is in: the sine has
  // the sign that its partner comes with
  constexpr int NP = MODE == kRunPairs ? 4 : 8;
  float c[NP], s[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    c[i] = 1.f, s[i] = 0.f;
    const int dim = MODE == kRunPairs ? d[0] + 2 * i : d[0] + i;
    if (dim < rot) {
      const bool second = MODE == kRunAlone && dim >= half;
      const int j = MODE == kRunPairs ? dim / 2 : second ? dim - half : dim;
      const float2_t cs = shared ? sines[mine0 + j] : turn4_of((double)pl.pos, p.inv_freq[j], p.scale);
      c[i] = cs[0], s[i] = MODE == kRunAlone && !second ? -cs[1] : cs[1];
    }
  }

  struct Loaded {
    EltVec<T, 8> x[RUNS], partner;
  };
  auto load = [&](const T *head, Loaded &x, bool turn) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
      load8<T, WHOLE, MODE != kRunAlone>(head + d[r], x.x[r]);
    if constexpr (MODE == kRunAlone)
      if (turn && turned) {
        if constexpr (WHOLE) { // (half is a multiple of 8)
          load8<T, true, false>(head + (d[0] < half ? d[0] + half : d[0] - half), x.partner);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int dim = d[0] + i;
            x.partner.v[i] = head[dim >= rot ? dim : dim < half ? dim + half : dim - half];
          }
        }
      }
  };
  auto values = [&](const Loaded &x, bool turn, float (&y)[RUNS][8]) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < RUNS; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y[r][i] = elt_to_f32(x.x[r].v[i]);
    if (!turn || !turned)
      return;
    if constexpr (MODE == kRunHalves) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = y[0][i], b = y[RUNS - 1][i];
        y[0][i] = turned4(a, c[i], b, -s[i]), y[RUNS - 1][i] = turned4(b, c[i], a, s[i]);
      }
    } else if constexpr (MODE == kRunPairs) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float a = y[0][2 * i], b = y[0][2 * i + 1];
        if (d[0] + 2 * i < rot)
          y[0][2 * i] = turned4(a, c[i], b, -s[i]), y[0][2 * i + 1] = turned4(b, c[i], a, s[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (d[0] + i < rot)
          y[0][i] = turned4(y[0][i], c[i], elt_to_f32(x.partner.v[i]), s[i]);
    }
  };

  // Heads are counted through q, k and v: a thread's are lane, lane + head_lanes, .. of them, so that
  // loads of all three are under way together.  A token without a page: its q alone.
  const int q_end = p.Hq, k_end = q_end + p.Hkv, end = pl.page < 0 ? q_end : k_end + p.Hkv;
  auto head_at = [&](int h) __attribute__((always_inline)) {
    return h < q_end   ? static_cast<const T *>(p.q) + t * p.q_st + h * p.q_sh
           : h < k_end ? static_cast<const T *>(p.k) + t * p.k_st + (h - q_end) * p.k_sh
                       : static_cast<const T *>(p.v) + t * p.v_st + (h - k_end) * p.v_sh;
  };
  auto turns = [&](int h) { return h < q_end ? pl.mine : h < k_end; };
  if constexpr (MODE == kRunAlone) // no blocks in q: a thread has whole pairs, so that q_out may be q
    if (p.Hq) {
      const T *const in = static_cast<const T *>(p.q) + t * p.q_st;
      T *const out = static_cast<T *>(p.q_out) + t * p.o_st;
      auto sine = [&](int j) __attribute__((always_inline)) {
        return shared ? sines[mine0 + j] : turn4_of((double)pl.pos, p.inv_freq[j], p.scale);
      };
      if constexpr (WHOLE) { // (half is a multiple of 8)
        const int rest = at.item - half / 8;
        const bool pair = rest < 0, turn = pair && pl.mine;
        const int a = pair ? 8 * at.item : rot + 8 * rest;
        if (a < p.head_dim) {
          float qc[8], qs[8];
          if (turn)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2_t cs = sine(a + i);
              qc[i] = cs[0], qs[i] = cs[1];
            }
          for (int h0 = at.lane; h0 < p.Hq; h0 += BATCH * p.head_lanes) {
            EltVec<T, 8> x[BATCH], z[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
              const int h = h0 + k * p.head_lanes;
              if (h < p.Hq) {
                load8<T, true, true>(in + h * p.q_sh + a, x[k]);
                if (pair)
                  load8<T, true, true>(in + h * p.q_sh + a + half, z[k]);
              }
            }
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
              const int h = h0 + k * p.head_lanes;
              if (h >= p.Hq)
                break;
              float y[2][8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float u = elt_to_f32(x[k].v[i]), w = pair ? elt_to_f32(z[k].v[i]) : 0.f;
                y[0][i] = turn ? turned4(u, qc[i], w, -qs[i]) : u, y[1][i] = turn ? turned4(w, qc[i], u, qs[i]) : w;
              }
              store8<T, true>(out + h * p.o_sh + a, y[0]);
              if (pair)
                store8<T, true>(out + h * p.o_sh + a + half, y[1]);
            }
          }
        }
      } else {
        for (int j = at.item; j < p.head_dim - half; j += p.items) {
          const bool pair = j < half, turn = pair && pl.mine;
          const int a = pair ? j : half + j;
          const float2_t cs = turn ? sine(j) : float2_t{1.f, 0.f};
          for (int h = at.lane; h < p.Hq; h += p.head_lanes) {
            const T *const from = in + h * p.q_sh + a;
            T *const to = out + h * p.o_sh + a;
            const T x = from[0], z = from[pair ? half : 0];
            const float u = elt_to_f32(x), w = elt_to_f32(z);
            to[0] = turn ? (T)turned4(u, cs[0], w, -cs[1]) : x;
            if (pair)
              to[half] = turn ? (T)turned4(w, cs[0], u, cs[1]) : z;
          }
        }
      }
    }
  const int64_t slot = pl.pos & ((1 << p.page_shift) - 1);
  for (int h0 = (MODE == kRunAlone ? q_end : 0) + at.lane; h0 < end; h0 += BATCH * p.head_lanes) {
    Loaded x[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
      if (const int h = h0 + k * p.head_lanes; h < end)
        load(head_at(h), x[k], turns(h));
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int h = h0 + k * p.head_lanes;
      if (h >= end)
        break;
      float y[RUNS][8];
      values(x[k], turns(h), y);
      if (MODE != kRunAlone && h < q_end) {
        T *const out = static_cast<T *>(p.q_out) + t * p.o_st + h * p.o_sh;
#pragma unroll
        for (int r = 0; r < RUNS; ++r)
          store8<T, WHOLE>(out + d[r], y[r]);
        continue;
      }
      const bool v = h >= k_end;
      const int hk = h - (v ? k_end : q_end);
      const BlockScales &bs = v ? args.vs : args.ks;
      uint8_t *const codes = v ? p.vc + pl.page * p.vc_sp + slot * p.vc_st + hk * p.vc_sh
                               : p.kc + pl.page * p.kc_sp + slot * p.kc_st + hk * p.kc_sh;
      uint8_t *const scales = bs.s + pl.page * bs.sp + slot * bs.st + hk * bs.sh;
      const float *const head_scale = v ? p.v_scale : p.k_scale;
      const float f = head_scale ? head_scale[hk] : 1.f;
#pragma unroll
      for (int r = 0; r < RUNS; ++r) {
        if (head_scale) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            y[r][i] = y[r][i] / f;
        }
        const uint32_t scale = block4_scale<NV>(block4_max<LANES>(y[r]), args.lo, args.hi);
        *reinterpret_cast<uint32_t *>(codes + d[r] / 2) = block4_codes<NV>(y[r], scale);
        if (d[r] / 8 % LANES == 0)
          scales[d[r] / (8 * LANES) * bs.sb] = scale;
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
  // Writes the values without a head's factor, where that takes no arithmetic.
  template <class O> __device__ __forceinline__ bool direct(O *) const { return false; }
};
template <bool NV> struct ReadItem<E2m1<NV>, 8> {
  uint32_t w, s;
  __device__ __forceinline__ void load(const uint8_t *head, int d, const BlockScales &bs, const uint8_t *scales) {
    w = *reinterpret_cast<const uint32_t *>(head + d / 2);
    s = scales[(d / (NV ? 16 : 32)) * bs.sb];
  }
  __device__ __forceinline__ void values(float (&y)[8]) const { codes4_f32<NV>(w, s, y); }
  // (the conversions round code * scale once; NV: fp16 holds the products, as Code4 takes them)
  template <class O> __device__ __forceinline__ bool direct(O *to) const {
    constexpr bool BF = std::is_same<O, __bf16>::value, HF = std::is_same<O, _Float16>::value;
    if constexpr ((BF && !NV) || HF) {
      uint32_t f = s << 23;
      if constexpr (NV)
        f = Code4<false, true>::factor(s, false);
      *reinterpret_cast<u32x4 *>(to) = Code4<BF, NV>::eight(w, f);
      return true;
    }
    return false;
  }
};

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
  // heads lane, lane + head_lanes, ..
  auto side = [&](const uint8_t *codes, int64_t sh, const BlockScales &bs, const float *head_scale, O *out,
                  int64_t oh) __attribute__((always_inline)) {
    const uint8_t *src = codes + at.lane * sh, *scales = bs.s + pl.page * bs.sp + slot * bs.st + at.lane * bs.sh;
    O *to = out + at.lane * oh + d;
    const int64_t step = p.head_lanes * sh, sstep = p.head_lanes * bs.sh, ostep = p.head_lanes * oh;
    for (int h0 = at.lane; h0 < p.Hkv; h0 += kHeadBatch * p.head_lanes) {
      ReadItem<C, VEC> x[kHeadBatch];
#pragma unroll
      for (int k = 0; k < kHeadBatch; ++k, src += step, scales += sstep)
        if (pl.page >= 0 && h0 + k * p.head_lanes < p.Hkv)
          x[k].load(src, d, bs, scales);
#pragma unroll
      for (int k = 0; k < kHeadBatch; ++k, to += ostep) {
        const int h = h0 + k * p.head_lanes;
        if (h >= p.Hkv)
          break;
        if (VEC == 8 && WHOLE && pl.page >= 0 && !head_scale && x[k].template direct<O>(to))
          continue;
        float y[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          y[i] = 0.f;
        if (pl.page >= 0) {
          x[k].values(y);
          if (head_scale) {
            const float f = head_scale[h];
#pragma unroll
            for (int i = 0; i < VEC; ++i)
              y[i] *= f;
          }
        }
        if constexpr (VEC == 8)
          store8<O, WHOLE>(to, y);
        else
          *to = (O)y[0];
      }
    }
  };
  side(p.kc + pl.page * p.kc_sp + slot * p.kc_st, p.kc_sh, p.ks, p.k_scale, static_cast<O *>(p.k) + t * p.k_st, p.k_sh);
  side(p.vc + pl.page * p.vc_sp + slot * p.vc_st, p.vc_sh, p.vs, p.v_scale, static_cast<O *>(p.v) + t * p.v_st, p.v_sh);
}

} // namespace txk
