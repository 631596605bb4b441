// Fragments of the paged attention's blocks (paged_attn.h): pages into LDS, K and V from there as
// MFMA operands, and the softmax between them.
#pragma once

#include "attn_fwd.h"
#include "page_rows.h"
#include "paged_sched.h"

namespace txk {

// s_waitcnt that no memory access of the compiler's crosses.
template <int N> __device__ __forceinline__ void paged_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void paged_lgkmcnt0() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
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
    return 16 * c >= row_bytes ? kOOB : page_run_row(row, run) * st + 16 * c;
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
    return 16 * c >= row_bytes ? P32::kOOB : page_run_row(row, run) * st + 16 * c;
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
  const int lr = (threadIdx.x & 63) / A::CPR;
  page_loads<U, A::R>(
      first, sd.run, [&](int row) __attribute__((always_inline)) { return resource(n + row); },
      [&](int u, const i32x4_t &rsrc, int r0) __attribute__((always_inline)) {
        if (r0 < 0 || (lr & ~(sd.run - 1)) == r0)
          paged_dma<NT>(off[u], rsrc, lds + (first + u) * 1024);
      });
}

} // namespace txk
