// Attention of new tokens over a paged cache (tx_cache.h).
//
// The G = Hq / Hkv query heads of one kv head read the same keys, so a sequence's new
// tokens make n G rows of one (sequence, kv head): row r is token r / G, head r % G.  A
// unit is a block of BM such rows; its keys are those between the first row's
// first and the last row's last, BN at a time.  Per block, on 32 rows a wave:
//   S^T = K . Q^T     32x32x16 MFMAs, A := K rows from LDS, B := Q rows, held in
//                     registers: lane l holds row l%32 and keys 8 (r/4) + 4 (l/32) + r%4 of
//                     each 32 of the block;
//   softmax           running maximum and sum in fp32 (base 2);
//   O^T += V^T . P^T  A := V columns by transposed LDS reads, B := P from the S^T
//                     registers, rounded to q's type (the matrix cores' operand; the sum of
//                     p is taken before that rounding).
// e4m3 caches are widened to q's type (exactly) between LDS and the matrix cores.
//
// Pages: a load into LDS takes 1 KiB, whole rows of one page, through a buffer
// resource made from the page's base by scalar instructions, so rows past the last
// key and pages that are not there come as zeros and no lane forms an address.  A lane
// holds each of 64 entries of the table row in turn.
//
// The lengths are known on the device only, and differ widely.  So the launch has one
// workgroup per place on the chip, all blocks of all units (kv heads outermost) are
// laid end to end, and each workgroup takes an equal run of them.  Parts of a unit go
// to the workspace, and the last workgroup to arrive joins them in order (so the
// result does not depend on which that is).
#pragma once

#include "attn_fwd.h"
#include "decode_i8.h"
#include "rotary.h"

namespace txk {

struct PagedAttnArgs {
  const void *q;
  const uint8_t *kc, *vc;
  const int32_t *table, *kv_len, *cu_q;
  const float *k_scale, *v_scale;
  void *o;
  float *lse;
  uint32_t *counters; // [grid]
  uint8_t *parts;     // [grid][2][A::PART]
  int64_t table_width, table_s;
  int64_t q_st, q_sh, o_st, o_sh;
  int64_t k_sp, k_st, k_sh, v_sp, v_st, v_sh; // bytes
  uint32_t pages, min_share;
  uint32_t g_mul, g_shift; // n / G = mulhi(n, g_mul) >> g_shift for n < 2^31 (G 1: g_mul 0)
  int32_t most; // keys that a table row has place for
  int32_t T, B, G, Hq, Hkv, head_dim, page_shift, causal, window;
  int32_t k_run, v_run; // rows of one resource
  float qk_scale;       // sm_scale / ln 2
};

// s_waitcnt that no memory access of the compiler's crosses.
template <int N> __device__ __forceinline__ void paged_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void paged_lgkmcnt0() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
__device__ __forceinline__ int lane_value(int v, int lane) {
  return __builtin_amdgcn_readlane(v, lane);
}
__device__ __forceinline__ int64_t lane_value64(int64_t v, int lane) {
  return (int64_t)(uint32_t)lane_value((int)v, lane) | (int64_t)lane_value((int)(v >> 32), lane) << 32;
}

// ---------------------------------------------------------------------------
// Fragments
// ---------------------------------------------------------------------------

// D: dims computed (heads of up to D); F8: the cache is e4m3; BN: keys of a block.
// LDS rows have a power of two of bytes (96 dims in rows of 128); 16-byte chunk c of row r
// lies at c ^ swizzle(r), so that the rows of one ds_read_b128 or transposed read fall on
// different banks.
template <int D_, bool BF, bool F8_, int BN_> struct PagedFrag {
  static constexpr int D = D_, BN = BN_, ROWS = 32;
  static constexpr bool F8 = F8_;
  static constexpr int ESZ = F8 ? 1 : 2;
  static constexpr int ROW = (D == 96 ? 128 : D) * ESZ, TILE = BN * ROW, CPR = ROW / 16;
  static constexpr int R = 1024 / ROW; // rows of a 1 KiB load
  static constexpr uint32_t kOOB = 0x80000000u;
  static_assert(D == 64 || D == 96 || D == 128 || D == 256, "head dims");
  static_assert(BN == 32 || BN == 64, "blocks");
  typedef AttnFwd<64, BF, 32, 64> X; // exchanges and MFMAs of the type
  typedef typename X::elt elt;
  typedef typename X::h8 h8;
  typedef typename X::h4 h4;
  typedef float f16v __attribute__((ext_vector_type(16)));
  typedef elt h2 __attribute__((ext_vector_type(2)));
  typedef int i32x2 __attribute__((ext_vector_type(2)));

  __device__ __forceinline__ static int kswz(int r) {
    return ROW == 64 ? (r >> 2) & 3 : ROW == 128 ? (r >> 1) & 7 : r & 15;
  }
  // 16-bit: 4 rows x 64 bytes of a pass; e4m3: 8 rows (keys 0-3 and 8-11 of 16) x 32 bytes.
  __device__ __forceinline__ static int vswz(int r) {
    if constexpr (F8)
      return ROW == 64    ? 2 * ((r >> 3) & 1)
             : ROW == 128 ? 2 * (((r >> 1) & 1) | ((r >> 2) & 2))
                          : 2 * ((r & 3) | ((r >> 1) & 4));
    else
      return ROW == 128 ? 4 * ((r >> 1) & 1) : 4 * (r & 3);
  }
  // 8 e4m3 values to q's type, exact.
  __device__ __forceinline__ static h8 widen(int lo, int hi) {
    h8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int w = i < 2 ? lo : hi;
      h2 t;
      if constexpr (BF)
        t = __builtin_bit_cast(h2, (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
      else
        t = __builtin_bit_cast(h2, (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
      r[2 * i] = t[0], r[2 * i + 1] = t[1];
    }
    return r;
  }

  // Lane offsets of the 1 KiB load `u` of a tile (row lane / CPR of it, at chunk position
  // lane % CPR), from the row that the load's resource begins with (one of every `run`).
  template <bool V>
  __device__ __forceinline__ static uint32_t offset(int u, uint32_t st, int run, int row_bytes) {
    const int lane = threadIdx.x & 63, row = R * u + lane / CPR, pos = lane % CPR;
    const int c = pos ^ (V ? vswz(row) : kswz(row));
    return 16 * c >= row_bytes ? kOOB : (uint32_t)(row & (run - 1)) * st + 16 * c;
  }

  // Per-lane LDS addresses of the fragment reads in a tile; the other fragments lie at
  // constants from these.
  //   K: key l%32, 16-byte chunk 2 c + l/32: dims 16 c + 8 (l/32) .. of MFMA c, or (e4m3) dims
  //     32 c + 16 (l/32) .., 8 each of MFMAs 2 c and 2 c + 1;
  //   V, dim block bd: the row and column that the lane gives a transposed read: 16-bit keys
  //     4 (l/32) + (l%16)/4 (and 8 further); e4m3 keys 4 (l/32) + 0..3 and + 8..11 by (l%16)/2.
  static constexpr int NK = F8 ? D / 32 : D / 16, NV = D / 32;
  struct Bases {
    uint32_t k[NK], v[NV];
  };
  __device__ __forceinline__ static void bases(uint32_t k_lds, uint32_t v_lds, Bases &bs) {
    const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5, L = lane & 15;
#pragma unroll
    for (int c = 0; c < NK; ++c)
      bs.k[c] = k_lds + r * ROW + (((2 * c + g) ^ kswz(r)) << 4);
#pragma unroll
    for (int bd = 0; bd < NV; ++bd) {
      const int d0 = 32 * bd + 16 * ((lane >> 4) & 1);
      if constexpr (F8) {
        const int j = L >> 1, key = 4 * g + (j & 3) + 8 * (j >> 2);
        bs.v[bd] = v_lds + key * ROW + (((d0 >> 4) ^ vswz(key)) << 4) + 8 * (L & 1);
      } else {
        const int d = d0 + 4 * (L & 3), key = 4 * g + (L >> 2);
        bs.v[bd] = v_lds + key * ROW + (((d >> 3) ^ vswz(key)) << 4) + (d & 7) * 2;
      }
    }
  }

  // Q rows as MFMA B operands in the order of K's dims.  scale < 0: the rows change their
  // sign, scale 0: they are zero, so that scores are taken times |scale| (or 1) > 0.
  struct QF {
    h8 v[D / 16];
  };
  __device__ __forceinline__ static int q_dim(int c) {
    const int g = (threadIdx.x & 63) >> 5;
    return F8 ? 32 * (c / 2) + 16 * g + 8 * (c % 2) : 16 * c + 8 * g;
  }
  __device__ __forceinline__ static void load_q(const void *row, int head_dim, QF &qf) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const int d = q_dim(c);
      qf.v[c] = *reinterpret_cast<const h8 *>(static_cast<const elt *>(row) + (d < head_dim ? d : 0));
    }
  }
  __device__ __forceinline__ static h8 settled(const h8 &q, bool live, float scale) {
    i32x4_t x = __builtin_bit_cast(i32x4_t, q);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = live && scale != 0.f ? x[i] ^ (scale < 0.f ? (int)0x80008000 : 0) : 0;
    return __builtin_bit_cast(h8, x);
  }
  __device__ __forceinline__ static void settle_q(bool live, int head_dim, float scale, QF &qf) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      qf.v[c] = settled(qf.v[c], live && q_dim(c) < head_dim, scale);
  }

  typedef f16v Scores[BN / 32];
  typedef f16v Acc[D / 32];
  typedef h8 PF[BN / 16];
  // K fragments of the tile at byte `at`.
  struct KF {
    i32x4_t v[BN / 32][NK];
  };
  __device__ __forceinline__ static void read_k(const Bases &bs, int at, KF &kf) {
    typedef __attribute__((address_space(3))) i32x4_t lds_i32x4;
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int b = 0; b < BN / 32; ++b)
        kf.v[b][c] = *(const lds_i32x4 *)(uintptr_t)(bs.k[c] + at + b * 32 * ROW);
  }
  __device__ __forceinline__ static void qk(const KF &kf, const QF &qf, f16v (&s)[BN / 32]) {
#pragma unroll
    for (int b = 0; b < BN / 32; ++b)
      s[b] = f16v{};
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int b = 0; b < BN / 32; ++b) { // independent sums side by side
        if constexpr (F8) {
          s[b] = X::mfma(widen(kf.v[b][c][0], kf.v[b][c][1]), qf.v[2 * c], s[b]);
          s[b] = X::mfma(widen(kf.v[b][c][2], kf.v[b][c][3]), qf.v[2 * c + 1], s[b]);
        } else {
          s[b] = X::mfma(__builtin_bit_cast(h8, kf.v[b][c]), qf.v[c], s[b]);
        }
      }
  }
  // V fragments of dim blocks b0 .. b0 + N - 1.
  template <int N> struct VF {
    i32x4_t v[N][BN / 16]; // e4m3: .xy
  };
  static constexpr int VN = NV < 4 ? NV : NV % 4 ? 3 : 4; // dim blocks read together
  template <int N>
  __device__ __forceinline__ static void read_v(const Bases &bs, int at, int b0, VF<N> &vf) {
#pragma unroll
    for (int bd = 0; bd < N; ++bd)
#pragma unroll
      for (int c = 0; c < BN / 16; ++c) {
        const uint32_t a = bs.v[b0 + bd] + at + c * 16 * ROW;
        if constexpr (F8) {
          typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
          const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(uintptr_t)a);
          vf.v[bd][c][0] = x[0], vf.v[bd][c][1] = x[1];
        } else {
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)a);
          const i16x4_t hi =
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)(a + 8 * ROW));
          vf.v[bd][c] =
              __builtin_bit_cast(i32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
      }
  }
  template <int N>
  __device__ __forceinline__ static void pv(const VF<N> &vf, int b0, const PF &pf, Acc &acc) {
#pragma unroll
    for (int c = 0; c < BN / 16; ++c)
#pragma unroll
      for (int bd = 0; bd < N; ++bd) { // independent sums side by side
        h8 x;
        if constexpr (F8)
          x = widen(vf.v[bd][c][0], vf.v[bd][c][1]);
        else
          x = __builtin_bit_cast(h8, vf.v[bd][c]);
        acc[b0 + bd] = X::mfma(x, pf[c], acc[b0 + bd]);
      }
  }

  // Scores of keys that the lane's row does not attend to (bit n of `seen`: it does to key n of
  // the block).
  __device__ __forceinline__ static void mask(f16v (&s)[BN / 32], uint64_t seen) {
    const uint64_t mine = seen >> (4 * ((threadIdx.x & 63) >> 5));
#pragma unroll
    for (int b = 0; b < BN / 32; ++b) {
      const uint32_t w = (uint32_t)(mine >> (32 * b));
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[b][r] = (w >> (8 * (r / 4) + r % 4)) & 1 ? s[b][r] : -INFINITY;
    }
  }

  // One block's softmax: s are its scores (times qk_scale > 0 they are base-2 exponents).
  // Updates the row's reference m (both lanes of a row hold the same), the lane's part of the sum
  // l, and acc; p as MFMA operands.  m follows the row's maximum only when that has grown past
  // it by 8, so acc is seldom rescaled; p is up to 2^8 then, in range in both types, and rounded by
  // the same relative half step.
  __device__ __forceinline__ static void softmax(f16v (&s)[BN / 32], float qk_scale,
                                                 f16v (&acc)[D / 32], float &m, float &l,
                                                 h8 (&pf)[BN / 16]) {
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < BN / 32; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        mx = fmaxf(mx, s[b][r]);
    mx = X::xmax(mx) * qk_scale;
    if (__builtin_expect(__any(mx > m + 8.f), 0)) {
      const float to = mx > m + 8.f ? mx : m;
      const float alpha = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.f : to));
      l *= alpha;
#pragma unroll
      for (int bd = 0; bd < D / 32; ++bd)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          acc[bd][r] *= alpha;
      m = to;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < BN / 32; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], qk_scale, -base));
        sum += s[b][r];
      }
    l += sum;
#pragma unroll
    for (int c = 0; c < BN / 16; ++c)
#pragma unroll
      for (int t = 0; t < 8; ++t)
        pf[c][t] = (elt)s[c / 2][8 * (c % 2) + t];
  }
  __device__ __forceinline__ static float row_sum(float v) { return X::xsum(v); }
  // acc as quads of 4 dims; where quad qd (dims 4 qd ..) of a row lies among them.
  typedef float f4v __attribute__((ext_vector_type(4)));
  static constexpr int QUADS = D / 8;
  __device__ __forceinline__ static f4v quad(const Acc &acc, int q) {
    return f4v{acc[q / 4][4 * (q % 4)], acc[q / 4][4 * (q % 4) + 1], acc[q / 4][4 * (q % 4) + 2],
               acc[q / 4][4 * (q % 4) + 3]};
  }
  __device__ __forceinline__ static int quad_at(int row, int qd) {
    return (qd >> 1) * 64 + row + 32 * (qd & 1);
  }
};

// The same on 16 rows a wave (decoding): 16x16x32 MFMAs, half the matrix and softmax work of 32 rows.
// Lane l holds of S^T row l%16 and keys 4 (l/16) + r of each 16; P's operand of 32 keys is those of
// two such blocks, and V's rows are read in that order.
template <int D_, bool BF, bool F8_, int BN_> struct PagedFrag16 {
  typedef PagedFrag<D_, BF, F8_, BN_> P32;
  static constexpr int D = D_, BN = BN_, ROWS = 16;
  static constexpr bool F8 = F8_;
  static constexpr int ESZ = P32::ESZ, ROW = P32::ROW, TILE = P32::TILE, CPR = P32::CPR, R = P32::R;
  typedef typename P32::X X;
  typedef typename X::elt elt;
  typedef typename X::h8 h8;
  typedef typename X::h4 h4;
  typedef float f4v __attribute__((ext_vector_type(4)));

  __device__ __forceinline__ static f4v mfma(const h8 &a, const h8 &b, const f4v &c) {
    if constexpr (BF)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  // A transposed read takes 16 rows x 32 bytes a half wave (keys 0-7), e4m3 16 rows (keys 0-7 and
  // 16-23) x 16 bytes.
  __device__ __forceinline__ static int vswz(int r) {
    if constexpr (F8)
      return ROW == 64    ? ((r >> 2) & 1) | ((r >> 3) & 2)
             : ROW == 128 ? ((r >> 1) & 3) | ((r >> 2) & 4)
                          : (r & 7) | ((r >> 1) & 8);
    else
      return ROW == 128 ? 2 * ((r >> 1) & 3) : 2 * (r & 7);
  }
  template <bool V>
  __device__ __forceinline__ static uint32_t offset(int u, uint32_t st, int run, int row_bytes) {
    const int lane = threadIdx.x & 63, row = R * u + lane / CPR, pos = lane % CPR;
    const int c = pos ^ (V ? vswz(row) : P32::kswz(row));
    return 16 * c >= row_bytes ? P32::kOOB : (uint32_t)(row & (run - 1)) * st + 16 * c;
  }

  //   K: key l%16, 16-byte chunk 4 c + l/16: dims 32 c + 8 (l/16) .. of MFMA c, or (e4m3) dims
  //     64 c + 16 (l/16) .., 8 each of MFMAs 2 c and 2 c + 1 (96 dims: as 128, with zeros);
  //   V, dim block bd of 16: 16-bit keys 4 (l/16) + (l%16)/4 (and 16 further); e4m3 keys
  //     4 (l/16) + 0..3 and + 16..19 by (l%16)/2.
  static constexpr int NK = F8 ? (D + 63) / 64 : D / 32, NQF = F8 ? 2 * NK : NK, NV = D / 16;
  struct Bases {
    uint32_t k[NK], v[NV];
  };
  __device__ __forceinline__ static void bases(uint32_t k_lds, uint32_t v_lds, Bases &bs) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int c = 0; c < NK; ++c)
      bs.k[c] = k_lds + r * ROW + (((4 * c + g) ^ P32::kswz(r)) << 4);
#pragma unroll
    for (int bd = 0; bd < NV; ++bd) {
      if constexpr (F8) {
        const int j = r >> 1, key = 4 * g + (j & 3) + 16 * (j >> 2);
        bs.v[bd] = v_lds + key * ROW + ((bd ^ vswz(key)) << 4) + 8 * (r & 1);
      } else {
        const int d = 16 * bd + 4 * (r & 3), key = 4 * g + (r >> 2);
        bs.v[bd] = v_lds + key * ROW + (((d >> 3) ^ vswz(key)) << 4) + (d & 7) * 2;
      }
    }
  }

  struct QF {
    h8 v[NQF];
  };
  __device__ __forceinline__ static int q_dim(int c) {
    const int g = (threadIdx.x & 63) >> 4;
    return F8 ? 64 * (c / 2) + 16 * g + 8 * (c % 2) : 32 * c + 8 * g;
  }
  __device__ __forceinline__ static void load_q(const void *row, int head_dim, QF &qf) {
#pragma unroll
    for (int c = 0; c < NQF; ++c) {
      const int d = q_dim(c);
      qf.v[c] = *reinterpret_cast<const h8 *>(static_cast<const elt *>(row) + (d < head_dim ? d : 0));
    }
  }
  __device__ __forceinline__ static void settle_q(bool live, int head_dim, float scale, QF &qf) {
#pragma unroll
    for (int c = 0; c < NQF; ++c)
      qf.v[c] = P32::settled(qf.v[c], live && q_dim(c) < head_dim, scale);
  }

  typedef f4v Scores[BN / 16];
  typedef f4v Acc[D / 16];
  struct KF {
    i32x4_t v[BN / 16][NK];
  };
  __device__ __forceinline__ static void read_k(const Bases &bs, int at, KF &kf) {
    typedef __attribute__((address_space(3))) i32x4_t lds_i32x4;
#pragma unroll
    for (int b = 0; b < BN / 16; ++b)
#pragma unroll
      for (int c = 0; c < NK; ++c)
        kf.v[b][c] = *(const lds_i32x4 *)(uintptr_t)(bs.k[c] + at + b * 16 * ROW);
  }
  __device__ __forceinline__ static void qk(const KF &kf, const QF &qf, Scores &s) {
#pragma unroll
    for (int b = 0; b < BN / 16; ++b)
      s[b] = f4v{};
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int b = 0; b < BN / 16; ++b) { // independent sums side by side
        if constexpr (F8) {
          s[b] = mfma(P32::widen(kf.v[b][c][0], kf.v[b][c][1]), qf.v[2 * c], s[b]);
          s[b] = mfma(P32::widen(kf.v[b][c][2], kf.v[b][c][3]), qf.v[2 * c + 1], s[b]);
        } else {
          s[b] = mfma(__builtin_bit_cast(h8, kf.v[b][c]), qf.v[c], s[b]);
        }
      }
  }
  template <int N> struct VF {
    i32x4_t v[N][BN / 32]; // e4m3: .xy
  };
  static constexpr int VN = NV < 8 ? NV : NV % 8 ? 6 : 8; // dim blocks read together
  __device__ __forceinline__ static void read_v(const Bases &bs, int at, int b0, VF<VN> &vf) {
#pragma unroll
    for (int bd = 0; bd < VN; ++bd)
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) {
        const uint32_t a = bs.v[b0 + bd] + at + c * 32 * ROW;
        if constexpr (F8) {
          typedef __attribute__((address_space(3))) typename P32::i32x2 lds_i32x2;
          const auto x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(uintptr_t)a);
          vf.v[bd][c][0] = x[0], vf.v[bd][c][1] = x[1];
        } else {
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)a);
          const i16x4_t hi =
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)(a + 16 * ROW));
          vf.v[bd][c] =
              __builtin_bit_cast(i32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
      }
  }
  typedef h8 PF[BN / 32];
  __device__ __forceinline__ static void pv(const VF<VN> &vf, int b0, const PF &pf, Acc &acc) {
#pragma unroll
    for (int c = 0; c < BN / 32; ++c)
#pragma unroll
      for (int bd = 0; bd < VN; ++bd) {
        h8 x;
        if constexpr (F8)
          x = P32::widen(vf.v[bd][c][0], vf.v[bd][c][1]);
        else
          x = __builtin_bit_cast(h8, vf.v[bd][c]);
        acc[b0 + bd] = mfma(x, pf[c], acc[b0 + bd]);
      }
  }
  __device__ __forceinline__ static void mask(Scores &s, uint64_t seen) {
    const uint64_t mine = seen >> (4 * ((threadIdx.x & 63) >> 4));
#pragma unroll
    for (int b = 0; b < BN / 16; ++b) {
      const uint32_t w = (uint32_t)(mine >> (16 * b));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        s[b][r] = (w >> r) & 1 ? s[b][r] : -INFINITY;
    }
  }
  // Across the lanes of a row (l%16).
  __device__ __forceinline__ static float row_max(float v) {
    v = X::xmax(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  __device__ __forceinline__ static float row_sum(float v) {
    v = X::xsum(v);
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  // As PagedFrag's.
  __device__ __forceinline__ static void softmax(Scores &s, float qk_scale, Acc &acc, float &m,
                                                 float &l, PF &pf) {
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < BN / 16; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        mx = fmaxf(mx, s[b][r]);
    mx = row_max(mx) * qk_scale;
    if (__builtin_expect(__any(mx > m + 8.f), 0)) {
      const float to = mx > m + 8.f ? mx : m;
      const float alpha = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.f : to));
      l *= alpha;
#pragma unroll
      for (int bd = 0; bd < NV; ++bd)
        acc[bd] *= alpha;
      m = to;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < BN / 16; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], qk_scale, -base));
        sum += s[b][r];
      }
    l += sum;
#pragma unroll
    for (int c = 0; c < BN / 32; ++c)
#pragma unroll
      for (int t = 0; t < 8; ++t)
        pf[c][t] = (elt)s[2 * c + t / 4][t % 4];
  }
  // acc as quads of 4 dims; where quad qd (dims 4 qd ..) of a row lies among them.
  static constexpr int QUADS = D / 16;
  __device__ __forceinline__ static f4v quad(const Acc &acc, int q) { return acc[q]; }
  __device__ __forceinline__ static int quad_at(int row, int qd) {
    return (qd >> 2) * 64 + row + 16 * (qd & 3);
  }
};

// ---------------------------------------------------------------------------
// Pages into LDS
// ---------------------------------------------------------------------------

// One wave's view of a table row: lane i holds entry `first` + i (-1: no page).
struct PageRow {
  const int32_t *row;
  uint32_t width, pages;
  int shift, first = 0, ids = -1;
  uint64_t holes = 0; // lanes without a page

  // Holds the entries of keys [n, n + 64); first their load (any entry past the row's end),
  // then their use.
  __device__ __forceinline__ void load(int n) {
    first = n >> shift;
    const uint32_t e = first + (threadIdx.x & 63);
    ids = row[e < width ? e : 0];
  }
  __device__ __forceinline__ void settle() {
    if (first + (threadIdx.x & 63) >= width || (uint32_t)ids >= pages)
      ids = -1;
    holes = __ballot(ids < 0);
  }
  __device__ __forceinline__ void hold(int n) {
    if (((n + 63) >> shift) >= first + 64) {
      load(n);
      settle();
    }
  }
  // Which of the BN keys from n on, before `end`, have a page.
  template <int BN> __device__ __forceinline__ uint64_t there(int n, int end) const {
    const uint64_t all = ~0ull >> (64 - BN);
    const int e0 = (n >> shift) - first, e1 = ((n + BN - 1) >> shift) - first;
    const uint64_t span = (~0ull >> (63 - (e1 - e0))) << e0;
    if (!(holes & span) && n + BN <= end)
      return all;
    const int key = n + (threadIdx.x & 63);
    const int id = __shfl(ids, ((key >> shift) - first) & 63);
    return __ballot(key < end && id >= 0) & all;
  }
};

// k or v of one kv head; run: rows that one resource covers, a power of two that divides
// a page and what a wave loads of a block.
struct PageSide {
  const uint8_t *base;
  int64_t sp, st;
  int run;
};

// 16 bytes a lane into LDS; NT: data that is read once.
template <bool NT>
__device__ __forceinline__ void paged_dma(uint32_t voff, const i32x4_t &rsrc, uint32_t lds) {
  if constexpr (NT)
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen nt lds" ::"v"(voff), "s"(rsrc), "{m0}"(lds)
                 : "memory");
  else
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "{m0}"(lds)
                 : "memory");
}

// Loads `first` .. first + U - 1 of the block of keys from n on into the tile at `lds`; rows
// from `end` on come as zeros.
template <class A, int U, bool NT>
__device__ __forceinline__ void issue_rows(const PageRow &pr, const PageSide &sd, int n, int end,
                                           int first, const uint32_t (&off)[U], uint32_t lds,
                                           int row_bytes) {
  auto resource = [&](int key) {
    const int id = lane_value(pr.ids, ((key >> pr.shift) - pr.first) & 63);
    const int slot = key & ((1 << pr.shift) - 1);
    const uint8_t *at = sd.base + (uint64_t)(uint32_t)id * (uint64_t)sd.sp +
                        (uint64_t)(uint32_t)slot * (uint64_t)sd.st;
    const int live = end - key < sd.run ? end - key : sd.run;
    const uint32_t bytes = (uint32_t)(live - 1) * (uint32_t)sd.st + (uint32_t)row_bytes;
    return make_rsrc(at, id < 0 || live <= 0 ? 0 : bytes);
  };
  // N resources of U / N loads each
  auto fast = [&](auto count) {
    constexpr int N = decltype(count)::value;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const i32x4_t rsrc = resource(n + A::R * (first + U / N * i));
#pragma unroll
      for (int u = U / N * i; u < U / N * (i + 1); ++u)
        paged_dma<NT>(off[u], rsrc, lds + (first + u) * 1024);
    }
  };
  if (sd.run >= U * A::R)
    fast(std::integral_constant<int, 1>());
  else if (U % 2 == 0 && 2 * sd.run >= U * A::R)
    fast(std::integral_constant<int, U % 2 ? 1 : 2>());
  else if (U % 4 == 0 && 4 * sd.run >= U * A::R)
    fast(std::integral_constant<int, U % 4 ? 1 : 4>());
  else { // pages of fewer rows; maybe fewer than a load has: the lanes of one at a time
    const int lr = (threadIdx.x & 63) / A::CPR;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma nounroll
      for (int r0 = 0; r0 < A::R; r0 += sd.run) {
        const i32x4_t rsrc = resource(n + A::R * (first + u) + r0);
        if (sd.run >= A::R || (lr & ~(sd.run - 1)) == r0)
          paged_dma<NT>(off[u], rsrc, lds + (first + u) * 1024);
      }
  }
}

// ---------------------------------------------------------------------------
// Which blocks are whose
// ---------------------------------------------------------------------------

// A unit of work: rows r0 .. r0 + rows - 1 of sequence b and kv head hk, whose tokens begin at
// row t0 of q and at position pos0, and of its steps those from s0 to s1.  Cut in parts,
// this one is `part`; part j is that of workgroup w0 + j, in its first place of the workspace, but
// part 0 in place slot0 (a workgroup's run has a cut unit at its beginning or at its end).
struct alignas(16) PagedUnit {
  int64_t pos0;
  int t0, r0, rows, hk, b, len, lo, hi; // keys [lo, hi)
  uint32_t s0, s1, parts, part, w0, slot0;
};
static_assert(sizeof(PagedUnit) == 64, "four 16-byte reads");

// What a unit's beginning and end cost, in steps.
constexpr uint32_t kSplitOverhead = 2, kRowsOverhead = 4;

// The token of a row.
__device__ __forceinline__ int paged_token(const PagedAttnArgs &p, int row) {
  return p.g_mul ? __umulhi((uint32_t)row, p.g_mul) >> p.g_shift : row;
}

// The keys [lo, hi) of rows [r0, r1) of a sequence of `len` keys whose first new token has
// position `at`.
__device__ __forceinline__ void paged_keys(const PagedAttnArgs &p, int64_t at, int len, int r0, int r1,
                                           int &lo, int &hi) {
  const int64_t last = at + paged_token(p, r1 - 1) + 1;
  const int64_t first = at + paged_token(p, r0) - p.window + 1;
  hi = len;
  if (p.causal && last < hi)
    hi = last < 0 ? 0 : (int)last;
  lo = p.window > 0 && first > 0 ? (int)(first < hi ? first : hi) : 0;
}

// Deals out the units.  Blocks of BN keys in steps of WPS blocks (those that the waves of a
// workgroup take side by side); a unit has one step at least, so that its rows are written, and
// begins with OV more that stand for what its beginning and end cost.  The first wave goes through this, a lane per sequence (64 at a time, in LDS) or block of rows; sums
// across lanes.
struct PagedSchedState {
  int64_t pos0[64];
  int t0[64], n[64], len[64];
  uint32_t cost[64];
  int cb, b, rb, hk;
  uint32_t S, share, pos, end, s0, w; // S: steps of a kv head
  PagedUnit unit[2]; // the current one and the next; rows 0: the end
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)(uint32_t)uniform((int)v) | (int64_t)uniform((int)(v >> 32)) << 32;
}

template <int BM, int BN, int WPS, uint32_t OV> struct PagedSched {
  const PagedAttnArgs &p;
  PagedSchedState &st;
  const int lane = threadIdx.x & 63;

  __device__ __forceinline__ PagedSched(const PagedAttnArgs &a, PagedSchedState &s) : p(a), st(s) {}

  // Inclusive sum over lanes, by DPP: rows of 16 lanes, then the rows.
  __device__ __forceinline__ static uint32_t upto(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false); // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false); // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
  }
  __device__ __forceinline__ static uint32_t steps_of(int lo, int hi) {
    if (hi <= lo)
      return 1;
    const int blocks = (int)(((uint32_t)hi + BN - 1) / BN) - lo / BN;
    return (blocks + WPS - 1) / WPS;
  }
  __device__ __forceinline__ uint32_t unit_steps(int64_t at, int len, int nr, int k) const {
    if (k * (int64_t)BM >= nr)
      return 0;
    int lo, hi;
    paged_keys(p, at, len, k * BM, nr - k * BM < BM ? nr : k * BM + BM, lo, hi);
    return OV + steps_of(lo, hi);
  }
  // The 64 sequences from `first` on; returns this lane's steps.
  __device__ __forceinline__ uint32_t load_chunk(int first) {
    const int q = first + lane;
    int n = 0, t0 = 0, len = 0;
    int64_t pos0 = 0;
    if (q < p.B) {
      const int raw = p.kv_len[q];
      if (p.cu_q) {
        const int a = p.cu_q[q], z = p.cu_q[q + 1];
        t0 = a > 0 ? a : 0;
        const int t1 = z < p.T ? z : p.T;
        n = t1 > t0 ? t1 - t0 : 0;
        pos0 = (int64_t)raw - z + t0;
      } else {
        t0 = q, n = 1, pos0 = (int64_t)raw - 1;
      }
      len = raw < 0 ? 0 : raw < p.most ? raw : p.most;
    }
    const int nr = n * p.G;
    uint32_t cost = 0;
    for (int k = 0; k < 2; ++k)
      if (nr <= 2 * BM)
        cost += unit_steps(pos0, len, nr, k);
    // sequences of many blocks of rows: a lane per block
    for (uint64_t big = __ballot(nr > 2 * BM); big; big &= big - 1) {
      const int from = __builtin_ctzll(big);
      const int64_t at = lane_value64(pos0, from);
      const int ln = lane_value(len, from), rows = lane_value(nr, from);
      uint32_t c = 0;
      for (int k = lane; k * (int64_t)BM < rows; k += 64)
        c += unit_steps(at, ln, rows, k);
      c = lane_value(upto(c), 63);
      if (lane == from)
        cost = c;
    }
    st.pos0[lane] = pos0, st.t0[lane] = t0, st.n[lane] = n, st.len[lane] = len;
    st.cost[lane] = cost;
    st.cb = first;
    return cost;
  }

  // The run of workgroup w of `grid`.
  __device__ __forceinline__ void init(uint32_t w, uint32_t grid) {
    uint32_t mine = 0;
    for (int c = 0; c < p.B; c += 64)
      mine += load_chunk(c);
    const uint32_t S = lane_value(upto(mine), 63), total = S * p.Hkv;
    uint32_t share = (total + grid - 1) / grid;
    share = share > p.min_share ? share : p.min_share;
    const uint64_t at = (uint64_t)share * w;
    st.w = w, st.S = S, st.share = share;
    st.pos = st.end = 0;
    if (at >= total)
      return;
    const uint32_t pos = (uint32_t)at;
    st.pos = pos, st.end = total - pos < share ? total : pos + share;
    const int hk = pos / S;
    uint32_t rem = pos - hk * S;
    st.hk = hk;
    int i = 0;
    // (The loops end at the last sequence and block also if lengths change meanwhile.)
    for (int c = 0; c < p.B; c += 64) {
      const uint32_t cost = p.B > 64 ? load_chunk(c) : st.cost[lane];
      const uint32_t upto_me = upto(cost), all = lane_value(upto_me, 63);
      if (rem < all) {
        i = __builtin_ctzll(__ballot(rem < upto_me));
        st.b = c + i;
        rem -= lane_value(upto_me, i) - lane_value(cost, i);
        break;
      }
      rem -= all;
    }
    // the block of rows
    const int rows = uniform(st.n[i]) * p.G, ln = uniform(st.len[i]);
    const int64_t p0 = uniform64(st.pos0[i]);
    int rb = 0;
    if (rows > BM)
      for (; (int64_t)rb * BM < rows; rb += 64) {
        const uint32_t c = unit_steps(p0, ln, rows, rb + lane);
        const uint32_t upto_me = upto(c), all = lane_value(upto_me, 63);
        if (rem < all) {
          const int j = __builtin_ctzll(__ballot(rem < upto_me));
          rem -= lane_value(upto_me, j) - lane_value(c, j);
          rb += j;
          break;
        }
        rem -= all;
      }
    st.rb = rb, st.s0 = rem;
  }

  // The next unit of the run, into `to`.
  __device__ __forceinline__ void get(PagedUnit &to) {
    const uint32_t end = uniform(st.end), share = uniform(st.share);
    uint32_t pos = uniform(st.pos), s0 = uniform(st.s0);
    int cb = uniform(st.cb), b = uniform(st.b), hk = uniform(st.hk), rb = uniform(st.rb);
    int my_n = st.n[lane], my_t0 = st.t0[lane], my_len = st.len[lane];
    int64_t my_pos0 = st.pos0[lane];
    PagedUnit u;
    u.rows = 0;
    while (pos < end && u.rows == 0) {
      const int i = b - cb, nr = lane_value(my_n, i) * p.G;
      u.b = b, u.hk = hk;
      u.t0 = lane_value(my_t0, i), u.len = lane_value(my_len, i), u.pos0 = lane_value64(my_pos0, i);
      u.r0 = rb * BM;
      const int rows = nr - u.r0 < BM ? nr - u.r0 : BM;
      paged_keys(p, u.pos0, u.len, u.r0, u.r0 + rows, u.lo, u.hi);
      const uint32_t cost = OV + steps_of(u.lo, u.hi);
      const uint32_t s1 = cost - s0 < end - pos ? cost : s0 + (end - pos);
      if (s1 > OV) {
        u.rows = rows;
        u.s0 = (s0 > OV ? s0 : OV) - OV, u.s1 = s1 - OV;
        u.parts = 1, u.part = 0, u.w0 = 0, u.slot0 = 0;
        if (u.s1 - u.s0 < cost - OV) {
          const uint32_t first = pos - s0;
          u.w0 = (first + OV) / share;
          u.parts = (first + cost - 1) / share - u.w0 + 1;
          u.part = uniform(st.w) - u.w0;
          u.slot0 = first < u.w0 * share ? 0 : 1;
        }
      }
      pos += s1 - s0, s0 = 0;
      if (pos >= end)
        break;
      if ((++rb) * (int64_t)BM >= nr) {
        rb = 0;
        uint64_t later = __ballot(st.cost[lane] > 0) & (i == 63 ? 0 : ~0ull << (i + 1));
        while (!later && hk < p.Hkv) {
          cb += 64;
          if (cb >= p.B)
            cb = 0, ++hk;
          later = __ballot((p.B > 64 ? load_chunk(cb) : st.cost[lane]) > 0);
          my_n = st.n[lane], my_t0 = st.t0[lane], my_len = st.len[lane], my_pos0 = st.pos0[lane];
        }
        if (!later || hk >= p.Hkv)
          pos = end;
        b = cb + (later ? __builtin_ctzll(later) : 0);
      }
    }
    st.pos = pos, st.s0 = 0, st.b = b, st.hk = hk, st.rb = rb;
    to = u;
  }
};

// The unit as scalars.
__device__ __forceinline__ PagedUnit paged_unit(const PagedUnit &s) {
  asm volatile("" ::: "memory"); // (read from LDS again)
  i32x4_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = reinterpret_cast<const i32x4_t *>(&s)[i];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    v[i / 4][i % 4] = uniform(v[i / 4][i % 4]);
  PagedUnit u;
  u.pos0 = (int64_t)(uint32_t)v[0][0] | (int64_t)v[0][1] << 32;
  u.t0 = v[0][2], u.r0 = v[0][3], u.rows = v[1][0], u.hk = v[1][1], u.b = v[1][2], u.len = v[1][3];
  u.lo = v[2][0], u.hi = v[2][1], u.s0 = v[2][2], u.s1 = v[2][3];
  u.parts = v[3][0], u.part = v[3][1], u.w0 = v[3][2], u.slot0 = v[3][3];
  return u;
}

// The kernel's arguments, read again from here on (they are not kept in registers through
// the loop before).
__device__ __forceinline__ const PagedAttnArgs &paged_args() {
  auto *a = (const __attribute__((address_space(4))) PagedAttnArgs *)
      __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *(const PagedAttnArgs *)a;
}

// Rows that belong to no sequence: zero.
template <class T> __device__ __forceinline__ void paged_zero_rows(const PagedAttnArgs &p) {
  if (!p.cu_q)
    return;
  int a = p.cu_q[0], z = p.cu_q[p.B];
  a = a < 0 ? 0 : a < p.T ? a : p.T;
  z = z < a ? a : z < p.T ? z : p.T;
  for (int64_t i = blockIdx.x; i < a + p.T - z; i += gridDim.x) {
    const int64_t t = i < a ? i : z + i - a;
    for (int h = 0; h < p.Hq; ++h) {
      for (int d = threadIdx.x; d < p.head_dim; d += blockDim.x)
        static_cast<T *>(p.o)[t * p.o_st + h * p.o_sh + d] = (T)0.f;
      if (threadIdx.x == 0 && p.lse)
        p.lse[t * p.Hq + h] = -INFINITY;
    }
  }
}

// A workgroup's place in the order of work: the 8 XCDs take contiguous runs.
__device__ __forceinline__ uint32_t paged_place() {
  const uint32_t n = gridDim.x, b = blockIdx.x;
  return b;
}

// One part's arrival: true in the last workgroup of the unit.  Data moves between
// workgroups with the SC1 policy only (decode_i8.h): stores are acknowledged before the count,
// loads follow it.
__device__ __forceinline__ bool paged_arrive(uint32_t *counter, uint32_t parts, int *flag) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t old =
        __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool last = old + 1 == parts;
    if (last)
      __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *reinterpret_cast<volatile int *>(flag) = last;
  }
  __syncthreads();
  const bool last = __builtin_amdgcn_readfirstlane(*reinterpret_cast<volatile int *>(flag));
  __syncthreads(); // the flag's next use
  return last;
}

// Joins (m1, l1, x1) to (m, l, x): sums relative to 2^m.
template <class V>
__device__ __forceinline__ void paged_join(float &m, float &l, V &x, float m1, float l1,
                                           const V &x1) {
  if (l1 == 0.f) // nothing (a NaN among the scores makes l NaN)
    return;
  const float to = fmaxf(m, m1);
  const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
  const float a1 = __builtin_amdgcn_exp2f(m1 - to);
  l = l * a + l1 * a1;
  x = x * a + x1 * a1;
  m = to;
}

typedef float f32x4v __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Few rows: the waves of a workgroup share out the keys
// ---------------------------------------------------------------------------

// LDS tiles that a wave has for K and for V: 16 KiB in all, or as much as its sums fill.
template <class A> constexpr int paged_split_slots() {
  constexpr int want = A::ROWS * A::D * 4 > 16384 ? A::ROWS * A::D * 4 : 16384;
  return want / (2 * A::TILE) > 0 ? want / (2 * A::TILE) : 1;
}
// 64 KiB of tiles leave a CU place for two workgroups.
template <class A> constexpr int paged_split_groups() {
  return 8 * paged_split_slots<A>() * A::TILE <= 65536 ? 2 : 1;
}

// 16 or 32 rows a unit (decoding, some drafted tokens).  Every wave goes through its own run of
// blocks, K and V each in one LDS tile of its own that is loaded again as soon as its
// fragments are in registers, with no barrier; at the end the four join in LDS.  Bound by
// memory: 8 waves a CU keep up to 16 KiB each in flight.
template <class A>
__global__ void __launch_bounds__(256, paged_split_groups<A>()) paged_attn_split_kernel(PagedAttnArgs args) {
  constexpr int D = A::D, BN = A::BN, ROWS = A::ROWS, U = A::TILE / 1024, NS = paged_split_slots<A>();
  typedef typename A::elt elt;
  typedef PagedSched<ROWS, BN, 4, kSplitOverhead> Sched;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4][2 * NS * A::TILE];
  __shared__ float ms[4][ROWS], ls[4][ROWS];
  __shared__ PagedSchedState st;
  __shared__ int flag;
  static_assert(ROWS * D * 4 <= 2 * NS * A::TILE, "a wave's sums fit its tiles");
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row_bytes = args.head_dim * A::ESZ;

  if (wave == 0) {
    Sched sched(args, st);
    sched.init(paged_place(), gridDim.x);
    sched.get(st.unit[0]);
  }
  __syncthreads();

  const uint32_t k_lds = lds_addr(smem[wave]), v_lds = k_lds + NS * A::TILE;
  typename A::Bases bs;
  A::bases(k_lds, v_lds, bs);
  uint32_t ko[U], vo[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    ko[u] = A::template offset<false>(u, (uint32_t)args.k_st, args.k_run, row_bytes);
    vo[u] = A::template offset<true>(u, (uint32_t)args.v_st, args.v_run, row_bytes);
  }
  const bool whole_loads = args.k_run >= A::R && args.v_run >= A::R;

  for (int turn = 0;; turn ^= 1) {
    const PagedAttnArgs &p = paged_args();
    const PagedUnit un = paged_unit(st.unit[turn]);
    if (un.rows <= 0)
      break;
    paged_vmcnt<0>(); // the loads below are counted
    // this wave's blocks
    int k0 = 0, k1 = 0;
    if (un.hi > un.lo) {
      const int first = un.lo / BN, last = (int)(((int64_t)un.hi + BN - 1) / BN);
      const int w0 = first + 4 * (int)un.s0;
      const int w1 = last - first < 4 * (int64_t)un.s1 ? last : first + 4 * (int)un.s1;
      const int q = (w1 - w0 + 3) / 4;
      k0 = w0 + wave * q < w1 ? w0 + wave * q : w1;
      k1 = k0 + q < w1 ? k0 + q : w1;
    }
    PageRow pr{p.table + un.b * p.table_s, (uint32_t)p.table_width, p.pages, p.page_shift};
    const PageSide sk{p.kc + un.hk * p.k_sh, p.k_sp, p.k_st, p.k_run};
    const PageSide sv{p.vc + un.hk * p.v_sh, p.v_sp, p.v_st, p.v_run};
    // The table, Q and the first blocks are under way together, and meanwhile the first wave
    // looks up the next unit.
    if (k0 < k1)
      pr.load(k0 * BN);
    const int r = lane % ROWS, rr = un.r0 + (r < un.rows ? r : 0);
    const int of = paged_token(p, rr), head = un.hk * p.G + rr - of * p.G;
    typename A::QF qf;
    A::load_q(static_cast<const elt *>(p.q) + (int64_t)(un.t0 + of) * p.q_st + head * p.q_sh,
              p.head_dim, qf);
    uint64_t here[NS + 1] = {}; // of blocks k .. k + NS
    if (k0 < k1) {
      pr.settle();
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (k0 + i < k1) {
          const int n = (k0 + i) * BN;
          pr.hold(n);
          here[i] = pr.template there<BN>(n, un.hi);
          issue_rows<A, U, true>(pr, sk, n, un.hi, 0, ko, k_lds + i * A::TILE, row_bytes);
          issue_rows<A, U, true>(pr, sv, n, un.hi, 0, vo, v_lds + i * A::TILE, row_bytes);
        }
    }
    if (wave == 0)
      Sched(p, st).get(st.unit[turn ^ 1]);
    int lo, hi; // of the lane's row
    paged_keys(p, un.pos0, un.len, rr, rr + 1, lo, hi);
    // keys that every row attends to
    int lo_all, hi_all, skip;
    paged_keys(p, un.pos0, un.len, un.r0, un.r0 + 1, skip, hi_all);
    paged_keys(p, un.pos0, un.len, un.r0 + un.rows - 1, un.r0 + un.rows, lo_all, skip);
    float scale = p.qk_scale * (p.k_scale ? p.k_scale[un.hk] : 1.f);
    A::settle_q(r < un.rows, p.head_dim, scale, qf);
    scale = scale == 0.f ? 1.f : fabsf(scale);
    float m = -INFINITY, l = 0.f;
    typename A::Acc acc = {};
    typename A::Scores s;
    auto iter = [&](int k, auto slot_c) {
      constexpr int SL = decltype(slot_c)::value;
      const int n0 = k * BN, na = n0 + NS * BN;
      const bool ahead = k + NS < k1;
      if (whole_loads && k + NS <= k1)
        paged_vmcnt<(2 * NS - 1) * U>(); // all after K_k
      else
        paged_vmcnt<0>();
      {
        typename A::KF kf;
        A::read_k(bs, SL * A::TILE, kf);
        paged_lgkmcnt0();
        if (ahead) {
          pr.hold(na);
          here[NS] = pr.template there<BN>(na, un.hi);
          issue_rows<A, U, true>(pr, sk, na, un.hi, 0, ko, k_lds + SL * A::TILE, row_bytes);
        }
        A::qk(kf, qf, s);
      }
      typename A::PF pf;
      const uint64_t all = ~0ull >> (64 - BN);
      if (here[0] != all || n0 < lo_all || n0 + BN > hi_all) {
        const int a = lo - n0 < 0 ? 0 : lo - n0, z = hi - n0 < 0 ? 0 : hi - n0;
        uint64_t seen = z < 64 ? (1ull << z) - 1 : ~0ull;
        seen &= a < 64 ? ~0ull << a : 0;
        A::mask(s, seen & here[0]);
      }
      A::softmax(s, scale, acc, m, l, pf);
      if (whole_loads && ahead)
        paged_vmcnt<(2 * NS - 1) * U>(); // all after V_k
      else
        paged_vmcnt<0>();
#pragma unroll
      for (int b0 = 0; b0 < A::NV; b0 += A::VN) {
        typename A::template VF<A::VN> vf;
        A::read_v(bs, SL * A::TILE, b0, vf);
        if (b0 + A::VN == A::NV) {
          paged_lgkmcnt0();
          if (ahead)
            issue_rows<A, U, true>(pr, sv, na, un.hi, 0, vo, v_lds + SL * A::TILE, row_bytes);
        }
        A::pv(vf, b0, pf, acc);
      }
#pragma unroll
      for (int i = 0; i < NS; ++i)
        here[i] = here[i + 1];
    };
    for (int k = k0; k < k1;) {
      iter(k++, std::integral_constant<int, 0>());
      if constexpr (NS >= 2)
        if (k < k1)
          iter(k++, std::integral_constant<int, 1>());
      if constexpr (NS == 4) {
        if (k < k1)
          iter(k++, std::integral_constant<int, 2>());
        if (k < k1)
          iter(k++, std::integral_constant<int, 3>());
      }
    }

    // The waves' sums: quads of 4 dims in lane order in each one's own tiles (all its loads
    // have landed).
    l = A::row_sum(l);
    const PagedAttnArgs &pe = paged_args();
    const PagedUnit ue = paged_unit(st.unit[turn]);
    const float vs = pe.v_scale ? pe.v_scale[ue.hk] : 1.f;
    if (k0 < k1) {
#pragma unroll
      for (int q = 0; q < A::QUADS; ++q)
        *reinterpret_cast<f32x4v *>(smem[wave] + (q * 64 + lane) * 16) = A::quad(acc, q);
    }
    if (lane < ROWS)
      ms[wave][lane] = m, ls[wave][lane] = l;
    __syncthreads();
    const int dq = pe.head_dim / 4, items = ue.rows * dq;
    const int64_t part_bytes = ROWS * (D + 2) * 4;
    uint8_t *const unit_parts = pe.parts;
    auto part_at = [&](uint32_t j) {
      const uint64_t slot = 2ull * (ue.w0 + j) + (j == 0 ? ue.slot0 : 0);
      return __builtin_amdgcn_make_buffer_rsrc(unit_parts + slot * part_bytes, 0, (int)part_bytes,
                                               0x00020000);
    };
    auto finish = [&](int row, int qd, float mm, float ll, f32x4v x) {
      const int ro = ue.r0 + row;
      const int of = paged_token(pe, ro), h = ue.hk * pe.G + ro - of * pe.G;
      const int64_t t = ue.t0 + of;
      const float f = ll == 0.f ? 0.f : vs / ll;
      typename A::h4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = (elt)(x[e] * f);
      *reinterpret_cast<typename A::h4 *>(static_cast<elt *>(pe.o) + t * pe.o_st + h * pe.o_sh +
                                          4 * qd) = y;
      if (qd == 0 && pe.lse)
        pe.lse[t * pe.Hq + h] = ll == 0.f ? -INFINITY : mm + __builtin_log2f(ll);
    };
    constexpr int kSC1 = 16;
    for (int it = tid; it < items; it += 256) {
      const int row = it / dq, qd = it % dq;
      float mm = -INFINITY, ll = 0.f;
      f32x4v x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int wv = 0; wv < 4; ++wv)
        paged_join(mm, ll, x, ms[wv][row], ls[wv][row],
                   *reinterpret_cast<const f32x4v *>(
                       smem[wv] + A::quad_at(row, qd) * 16));
      if (ue.parts == 1) {
        finish(row, qd, mm, ll, x);
      } else {
        const auto mine = part_at(ue.part);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4_t, x), mine,
                                               (row * D + 4 * qd) * 4, 0, kSC1);
        if (qd == 0) {
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(mm), mine, (ROWS * D + row) * 4, 0,
                                                kSC1);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(ll), mine,
                                                (ROWS * D + ROWS + row) * 4, 0, kSC1);
        }
      }
    }
    __syncthreads(); // the tiles' and ms' next use
    if (ue.parts == 1 || !paged_arrive(&pe.counters[ue.w0], ue.parts, &flag))
      continue;
    // Last: all parts, in order.  Threads past one set of items take other parts.
    const int groups = items < 256 ? 256 / items : 1;
    for (int base = 0; base < items; base += 256) {
      const int gi = items < 256 ? tid / items : 0, it = items < 256 ? tid % items : base + tid;
      const bool on = gi < groups && it < items;
      const int row = on ? it / dq : 0, qd = on ? it % dq : 0;
      float mm = -INFINITY, ll = 0.f;
      f32x4v x = {0.f, 0.f, 0.f, 0.f};
      constexpr int NJ = 8; // parts in flight
      for (uint32_t j0 = gi; j0 < ue.parts; j0 += NJ * groups) {
        float pm[NJ], pl[NJ];
        i32x4_t px[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint32_t jj = j0 + j * groups;
          pm[j] = -INFINITY, pl[j] = 0.f;
          if (on && jj < ue.parts) {
            const uint64_t slot = 2ull * (ue.w0 + jj) + (jj == 0 ? ue.slot0 : 0);
            const auto all = __builtin_amdgcn_make_buffer_rsrc(unit_parts, 0, 0x7fffffff, 0x00020000);
            const int at = (int)(slot * part_bytes);
            px[j] = __builtin_bit_cast(
                i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(all, at + (row * D + 4 * qd) * 4, 0, kSC1));
            pm[j] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(all, at + (ROWS * D + row) * 4, 0, kSC1));
            pl[j] = __int_as_float(
                __builtin_amdgcn_raw_buffer_load_b32(all, at + (ROWS * D + ROWS + row) * 4, 0, kSC1));
          }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          paged_join(mm, ll, x, pm[j], pl[j], __builtin_bit_cast(f32x4v, px[j]));
      }
      if (groups > 1) {
        f32x4v *const xs = reinterpret_cast<f32x4v *>(smem[0]);
        float *const mls = reinterpret_cast<float *>(smem[0] + 4096);
        xs[tid] = x;
        mls[tid] = mm, mls[256 + tid] = ll;
        __syncthreads();
        if (tid < items) {
          for (int k = 1; k < groups; ++k)
            paged_join(mm, ll, x, mls[k * items + tid], mls[256 + k * items + tid],
                       xs[k * items + tid]);
          finish(row, qd, mm, ll, x);
        }
        __syncthreads();
      } else if (on) {
        finish(row, qd, mm, ll, x);
      }
    }
  }
  paged_zero_rows<elt>(args);
}

// ---------------------------------------------------------------------------
// Many rows: the waves of a workgroup share the keys
// ---------------------------------------------------------------------------

// 128 rows a unit, 32 a wave (chunks of a prompt).  K and V have two LDS slots each.  A block has
// two barriers: after the first K_k is whole (and V_{k-1}'s slot free, for V_{k+1}), after the second
// V_k is (and K_k's slot free, for K_{k+2}), so that loads have about two blocks' time to land.  All
// of K's fragments are under way before the first of their MFMAs, all of V's before the softmax.  The
// matrix cores and the softmax overlap between the workgroups of a CU.
template <class A> constexpr int paged_rows_groups() { return A::D > 128 ? 1 : A::D > 64 ? 2 : 3; }

template <class A>
__global__ void __launch_bounds__(256, paged_rows_groups<A>()) paged_attn_rows_kernel(PagedAttnArgs args) {
  constexpr int D = A::D, BN = A::BN, U = A::TILE / 4096; // loads of a wave
  typedef typename A::elt elt;
  typedef PagedSched<128, BN, 1, kRowsOverhead> Sched;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * A::TILE];
  __shared__ PagedSchedState st;
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row_bytes = args.head_dim * A::ESZ;

  if (wave == 0) {
    Sched sched(args, st);
    const uint32_t n = gridDim.x, b = blockIdx.x;
    sched.init(n % 8 == 0 ? (b % 8) * (n / 8) + b / 8 : b, n);
    sched.get(st.unit[0]);
  }
  __syncthreads();

  const uint32_t k_lds = lds_addr(smem), v_lds = k_lds + 2 * A::TILE;
  typename A::Bases bs;
  A::bases(k_lds, v_lds, bs);
  uint32_t ko[U], vo[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    ko[u] = A::template offset<false>(U * wave + u, (uint32_t)args.k_st, args.k_run, row_bytes);
    vo[u] = A::template offset<true>(U * wave + u, (uint32_t)args.v_st, args.v_run, row_bytes);
  }

  const bool whole_loads = args.k_run >= A::R && args.v_run >= A::R;

  for (int turn = 0;; turn ^= 1) {
    const PagedAttnArgs &p = paged_args();
    const PagedUnit un = paged_unit(st.unit[turn]);
    if (un.rows <= 0)
      break;
    paged_vmcnt<0>(); // the loads below are counted
    int k0 = 0, k1 = 0;
    if (un.hi > un.lo) {
      const int first = un.lo / BN, last = (int)(((int64_t)un.hi + BN - 1) / BN);
      k0 = first + (int)un.s0;
      k1 = first + (int)un.s1 < last ? first + (int)un.s1 : last;
    }
    PageRow pr{p.table + un.b * p.table_s, (uint32_t)p.table_width, p.pages, p.page_shift};
    const PageSide sk{p.kc + un.hk * p.k_sh, p.k_sp, p.k_st, p.k_run};
    const PageSide sv{p.vc + un.hk * p.v_sh, p.v_sp, p.v_st, p.v_run};
    uint64_t here[3] = {}; // of blocks k, k + 1, k + 2
    auto issue_k = [&](int k, int slot) {
      issue_rows<A, U, false>(pr, sk, k * BN, un.hi, U * wave, ko, k_lds + slot * A::TILE, row_bytes);
    };
    auto issue_v = [&](int k, int slot) {
      issue_rows<A, U, false>(pr, sv, k * BN, un.hi, U * wave, vo, v_lds + slot * A::TILE, row_bytes);
    };
    // The table, Q and the first blocks are under way together, and meanwhile the first wave
    // looks up the next unit.
    if (k0 < k1)
      pr.load(k0 * BN);
    const bool busy = un.rows > 32 * wave;
    const int r = 32 * wave + (lane & 31), rr = un.r0 + (r < un.rows ? r : 0);
    const int of = paged_token(p, rr), head = un.hk * p.G + rr - of * p.G;
    typename A::QF qf;
    A::load_q(static_cast<const elt *>(p.q) + (int64_t)(un.t0 + of) * p.q_st + head * p.q_sh,
              p.head_dim, qf);
    if (k0 < k1) {
      pr.settle();
      here[0] = pr.template there<BN>(k0 * BN, un.hi);
      issue_k(k0, 0);
      issue_v(k0, 0);
      if (k0 + 1 < k1) {
        pr.hold((k0 + 1) * BN);
        here[1] = pr.template there<BN>((k0 + 1) * BN, un.hi);
        issue_k(k0 + 1, 1);
      }
    }
    if (wave == 0)
      Sched(p, st).get(st.unit[turn ^ 1]);
    int lo, hi; // of the lane's row
    paged_keys(p, un.pos0, un.len, rr, rr + 1, lo, hi);
    // of the wave's rows: keys that all attend to, and keys that any does
    int lo_all = 0, hi_all = 0, lo_any = 0, hi_any = 0;
    if (busy) {
      const int a = un.r0 + 32 * wave, z = un.r0 + (un.rows < 32 * wave + 32 ? un.rows : 32 * wave + 32);
      paged_keys(p, un.pos0, un.len, a, a + 1, lo_any, hi_all);
      paged_keys(p, un.pos0, un.len, z - 1, z, lo_all, hi_any);
    }
    auto live = [&](int k) { return busy && k * BN < hi_any && k * BN + BN > lo_any; };
    float scale = p.qk_scale * (p.k_scale ? p.k_scale[un.hk] : 1.f);
    A::settle_q(r < un.rows, p.head_dim, scale, qf);
    scale = scale == 0.f ? 1.f : fabsf(scale);
    float m = -INFINITY, l = 0.f;
    typename A::Acc acc = {};
    typename A::Scores s;
    paged_vmcnt<0>();
    __syncthreads();
    auto iter = [&](int k, auto slot_c) {
      constexpr int SL = decltype(slot_c)::value;
      const int n0 = k * BN;
      const bool on = live(k);
      if (k + 1 < k1)
        issue_v(k + 1, 1 - SL);
      if (on) {
        typename A::KF kf;
        A::read_k(bs, SL * A::TILE, kf);
        __builtin_amdgcn_sched_barrier(0);
        A::qk(kf, qf, s);
      }
      if (whole_loads && k + 1 < k1)
        paged_vmcnt<2 * U>(); // all after V_k
      else
        paged_vmcnt<0>();
      __syncthreads();
      if (k + 2 < k1) {
        pr.hold((k + 2) * BN);
        here[2] = pr.template there<BN>((k + 2) * BN, un.hi);
        issue_k(k + 2, SL);
      }
      if (on) {
        typename A::template VF<A::NV> vf;
        A::read_v(bs, SL * A::TILE, 0, vf);
        __builtin_amdgcn_sched_barrier(0);
        const uint64_t all = ~0ull >> (64 - BN);
        if (here[0] != all || n0 < lo_all || n0 + BN > hi_all) {
          const int a = lo - n0 < 0 ? 0 : lo - n0, z = hi - n0 < 0 ? 0 : hi - n0;
          uint64_t seen = z < 64 ? (1ull << z) - 1 : ~0ull;
          seen &= a < 64 ? ~0ull << a : 0;
          A::mask(s, seen & here[0]);
        }
        typename A::PF pf;
        A::softmax(s, scale, acc, m, l, pf);
        A::pv(vf, 0, pf, acc);
      }
      here[0] = here[1], here[1] = here[2];
      if (whole_loads && k + 2 < k1)
        paged_vmcnt<2 * U>(); // all after K_{k+1}
      else
        paged_vmcnt<0>();
      __syncthreads();
    };
    for (int k = k0; k < k1;) {
      iter(k++, std::integral_constant<int, 0>());
      if (k < k1)
        iter(k++, std::integral_constant<int, 1>());
    }

    l = A::X::xsum(l);
    const PagedAttnArgs &pe = paged_args();
    const PagedUnit ue = paged_unit(st.unit[turn]);
    __syncthreads(); // (the first wave will write the unit after the next there)
    const float vs = pe.v_scale ? pe.v_scale[ue.hk] : 1.f;
    const int r_e = 32 * wave + (lane & 31), rr_e = ue.r0 + (r_e < ue.rows ? r_e : 0);
    const bool busy_e = ue.rows > 32 * wave;
    const int of_e = paged_token(pe, rr_e), head_e = ue.hk * pe.G + rr_e - of_e * pe.G;
    const int64_t tok_e = ue.t0 + of_e;
    const int64_t part_bytes = 128 * (D + 2) * 4;
    constexpr int kSC1 = 16;
    if (ue.parts > 1) {
      // (lane order: quads of a wave side by side)
      const uint64_t slot = 2ull * (ue.w0 + ue.part) + (ue.part == 0 ? ue.slot0 : 0);
      const auto mine = __builtin_amdgcn_make_buffer_rsrc(pe.parts + slot * part_bytes, 0,
                                                          (int)part_bytes, 0x00020000);
      if (busy_e) {
#pragma unroll
        for (int q = 0; q < D / 8; ++q)
          __builtin_amdgcn_raw_buffer_store_b128(
              __builtin_bit_cast(i32x4_t, f32x4v{acc[q / 4][4 * (q % 4)], acc[q / 4][4 * (q % 4) + 1],
                                                 acc[q / 4][4 * (q % 4) + 2],
                                                 acc[q / 4][4 * (q % 4) + 3]}),
              mine, ((wave * (D / 8) + q) * 64 + lane) * 16, 0, kSC1);
        if (g == 0) {
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(m), mine, (128 * D + r_e) * 4, 0, kSC1);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(l), mine, (128 * D + 128 + r_e) * 4, 0,
                                                kSC1);
        }
      }
      if (!paged_arrive(&pe.counters[ue.w0], ue.parts, &flag))
        continue;
      if (busy_e) {
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (int bd = 0; bd < D / 32; ++bd)
          acc[bd] = typename A::f16v{};
        for (uint32_t j = 0; j < ue.parts; ++j) {
          const uint64_t from = 2ull * (ue.w0 + j) + (j == 0 ? ue.slot0 : 0);
          const auto part = __builtin_amdgcn_make_buffer_rsrc(pe.parts + from * part_bytes, 0,
                                                              (int)part_bytes, 0x00020000);
          i32x4_t x[D / 8];
#pragma unroll
          for (int q = 0; q < D / 8; ++q)
            x[q] = __builtin_bit_cast(
                i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                             part, ((wave * (D / 8) + q) * 64 + lane) * 16, 0, kSC1));
          const float m1 = __int_as_float(
              __builtin_amdgcn_raw_buffer_load_b32(part, (128 * D + r_e) * 4, 0, kSC1));
          const float l1 = __int_as_float(
              __builtin_amdgcn_raw_buffer_load_b32(part, (128 * D + 128 + r_e) * 4, 0, kSC1));
          if (l1 == 0.f)
            continue;
          const float to = fmaxf(m, m1);
          const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
          const float a1 = __builtin_amdgcn_exp2f(m1 - to);
          l = l * a + l1 * a1;
          m = to;
#pragma unroll
          for (int q = 0; q < D / 8; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[q / 4][4 * (q % 4) + e] =
                  acc[q / 4][4 * (q % 4) + e] * a + __int_as_float(x[q][e]) * a1;
        }
      }
    }
    if (r_e < ue.rows) {
      const float f = l == 0.f ? 0.f : vs / l;
      elt *const orow = static_cast<elt *>(pe.o) + tok_e * pe.o_st + head_e * pe.o_sh;
#pragma unroll
      for (int q = 0; q < D / 8; ++q) {
        const int d = 32 * (q / 4) + 8 * (q % 4) + 4 * g;
        typename A::h4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[e] = (elt)(acc[q / 4][4 * (q % 4) + e] * f);
        if (d < pe.head_dim)
          *reinterpret_cast<typename A::h4 *>(orow + d) = y;
      }
      if (g == 0 && pe.lse)
        pe.lse[tok_e * pe.Hq + head_e] = l == 0.f ? -INFINITY : m + __builtin_log2f(l);
    }
  }
  paged_zero_rows<elt>(args);
}

} // namespace txk
