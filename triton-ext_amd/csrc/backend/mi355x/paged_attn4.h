// Attention of new tokens over a paged cache held in 4 bits (tx_cache4.h).  Units of work, their
// schedule, softmax, masks and joins are those of paged_attn.h; keys and values come otherwise.
//
// A row of codes is 16 .. 128 bytes, a quarter of what LDS tiles of 16-bit pages are made for, so
// they are loaded into registers, straight from the pages: of 16 keys, lane (m, g) takes the
// g-th quarter of key m's row (of 256 dims: one 16-byte piece of each half).  A piece is 8 bytes
// (heads of up to 64) or 16 (32 dims: one or two blocks), so the conversion to 16 bits needs one or
// two factors; the scales come as dwords of four keys and reach their lanes by ds_bpermute.
//
// Codes become the 16-bit type that q is in, which holds every code under an e8m0 scale of its range
// exactly; under e4m3 scales fp16, which holds all of their products exactly too and, unlike bf16, is
// multiplied two at a time.
//
// K: S^T = K . Q^T does not ask in which order dims are summed.  With m = lane % 16 the lane's
// dims are an operand of the 16x16x32 MFMAs as they stand, Q is loaded in the same order, and K
// never goes through LDS.  V: the product needs several keys of one dim in a lane, so with m =
// lane / 4 its values are written into an LDS tile of 16-bit rows and read transposed.
//
// Lanes of keys that are not there read page 0 (there is one, or nothing is read); whatever it
// holds, their scores are -inf and their V finite: a scale that may make no number is taken as 0
// in V, and the key's score is NaN instead for the rows that attend to it.
#pragma once

#include "cache4.h"
#include "cache4_rows.h"
#include "paged_attn.h"

namespace txk {

struct Paged4Args {
  PagedAttnArgs a; // (first: paged_args() reads it)
  BlockScales ks, vs;
  int32_t packed; // the scales of 4 keys from a multiple of 4 on are an aligned dword
};
__device__ __forceinline__ const Paged4Args &paged4_args() {
  return reinterpret_cast<const Paged4Args &>(paged_args());
}

// x, as something that the compiler does not form other values from outside the loop.
__device__ __forceinline__ uint32_t here_only(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// What a lane holds of one key's K or V row, in the order of its quarter g: KW dwords of 8 dims, under SB
// block scales.
template <int D, bool NV> struct Piece4 {
  static constexpr int KW = D == 64 ? 2 : D == 256 ? 8 : 4;
  static constexpr int SB = D == 64 ? 1 : (D == 256 ? 2 : 1) * (NV ? 2 : 1);
  uint32_t w[KW];

  // The dims of dword c, the scale that is theirs, and the block of scale j.
  __device__ __forceinline__ static constexpr int dim(int c, int g) {
    return D == 64 ? 16 * g + 8 * c : 128 * (c / 4) + 32 * g + 8 * (c % 4);
  }
  // Dword c's place in a 16-bit row of 16-byte chunks, from dword 0's: bits that dword 0's chunk (16 g,
  // or 4 g chunks) has not set, so that a swizzle of the chunks commutes with it.
  __device__ __forceinline__ static constexpr uint32_t at(int c) { return 2 * dim(c, 0); }
  __device__ __forceinline__ static constexpr int scale_of(int c) {
    return D == 64 ? 0 : NV ? c / 2 : c / 4;
  }
  __device__ __forceinline__ static constexpr int block_of(int j, int g) {
    if (D == 64)
      return NV ? g : g / 2;
    return NV ? 8 * (j / 2) + 2 * g + j % 2 : 4 * j + g;
  }
};

// One wave's view of a table row, and where an entry's page begins in the arrays: 0, 1: codes and scales of
// K, 2, 3: of V (page 0 where there is none).  KEPT: found for all 64 entries at once (a wave that loads
// all of a block by itself), else when asked for (8 registers less).
template <bool KEPT> struct PageRow4 : PageRow {
  uint64_t at[KEPT ? 4 : 1];

  template <int I> __device__ __forceinline__ static uint64_t stride() {
    const Paged4Args &p = paged4_args();
    return (uint64_t)(I == 0 ? p.a.k_sp : I == 1 ? p.ks.sp : I == 2 ? p.a.v_sp : p.vs.sp);
  }
  __device__ __forceinline__ void settle() {
    PageRow::settle();
    if constexpr (KEPT) {
      const uint64_t id = ids < 0 ? 0 : ids;
      at[0] = id * stride<0>(), at[1] = id * stride<1>(), at[2] = id * stride<2>(), at[3] = id * stride<3>();
    }
  }
  __device__ __forceinline__ void hold(int n) {
    if (((n + 63) >> shift) >= first + 64) {
      load(n);
      settle();
    }
  }
  // Of entry `e` of those held, the same for all lanes; or each lane its own.
  template <int I> __device__ __forceinline__ uint64_t place(int e) const {
    if constexpr (KEPT)
      return (uint64_t)lane_value64(at[I], e & 63);
    const int id = lane_value(ids, e & 63);
    return (uint64_t)(uint32_t)(id < 0 ? 0 : id) * stride<I>();
  }
  template <int I> __device__ __forceinline__ uint64_t places(int e) const {
    if constexpr (KEPT)
      return (uint64_t)(uint32_t)__shfl((int)at[I], e & 63) | (uint64_t)(uint32_t)__shfl((int)(at[I] >> 32), e & 63) << 32;
    const int id = __shfl(ids, e & 63);
    return (uint64_t)(uint32_t)(id < 0 ? 0 : id) * stride<I>();
  }
};

// Where lane (m, g) finds its pieces of K (V: of V) of 16 keys: the codes of a head, which are
// uniform, and the lane's offsets from the first key, of 32 bits.  Pieces past head_dim are those of
// its beginning (Q is 0 there; V's are not stored).
template <int D, bool NV, bool V> struct Side4 {
  typedef Piece4<D, NV> P;
  const uint8_t *codes;
  uint32_t st;
  uint32_t off[D == 256 ? 2 : 1];

  __device__ __forceinline__ Side4(const Paged4Args &p, int hk, int m, int g) {
    codes = (V ? p.a.vc : p.a.kc) + hk * (V ? p.a.v_sh : p.a.k_sh);
    st = (uint32_t)(V ? p.a.v_st : p.a.k_st);
    const uint32_t row = p.a.page_shift >= 4 ? m : m & ((1 << p.a.page_shift) - 1);
    const int bytes = p.a.head_dim / 2;
#pragma unroll
    for (int i = 0; i < (D == 256 ? 2 : 1); ++i) {
      const int o = D == 64 ? 8 * g : 64 * i + 16 * g;
      off[i] = row * st + (o < bytes ? o : 0);
    }
  }
  template <bool NT, class W> __device__ __forceinline__ static W take(const uint8_t *p) {
    if constexpr (NT)
      return __builtin_nontemporal_load(reinterpret_cast<const W *>(p));
    else
      return *reinterpret_cast<const W *>(p);
  }
  template <bool NT> __device__ __forceinline__ void read(const uint8_t *c, P &x) const {
    typedef uint32_t w2 __attribute__((ext_vector_type(2)));
    typedef uint32_t w4 __attribute__((ext_vector_type(4)));
    if constexpr (D == 64) {
      const w2 v = take<NT, w2>(c + off[0]);
      x.w[0] = v[0], x.w[1] = v[1];
    } else {
#pragma unroll
      for (int i = 0; i < P::KW / 4; ++i) {
        const w4 v = take<NT, w4>(c + off[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x.w[4 * i + e] = v[e];
      }
    }
  }
  // The pieces of N runs of 16 keys from n on, a multiple of 16 N; m is the lane's row again.  NT: data
  // that is read once.
  template <bool NT, int N, class Row>
  __device__ __forceinline__ void load(const Row &pr, int n, int m, P (&x)[N]) const {
    if (pr.shift >= 4) { // a run lies in one page
      const uint8_t *c;
#pragma unroll
      for (int b = 0; b < N; ++b) {
        if (b == 0 || pr.shift < 5) {
          const int key = n + 16 * b;
          const uint64_t slot = key & ((1 << pr.shift) - 1);
          c = codes + pr.template place<V ? 2 : 0>((key >> pr.shift) - pr.first) + slot * st;
        } else {
          c += 16ull * st;
        }
        read<NT>(c, x[b]);
      }
    } else {
#pragma unroll
      for (int b = 0; b < N; ++b)
        read<NT>(codes + pr.template places<V ? 2 : 0>(((n + 16 * b + m) >> pr.shift) - pr.first), x[b]);
    }
  }
};

// The block scales of KEYS keys' K and V: a lane holds dwords of 4 keys of a block each, in the order
// [K, V][block][4 keys], which one or two loads of whole lines bring (a byte a lane and key took the
// same memory 98 us where this takes 88: 4 sequences of up to 131072); the lanes that convert fetch their
// byte from there.
// ALIKE: the lane has the same piece of K and of V.
template <int D, bool NV, int KEYS, bool ALIKE> struct Scales4 {
  typedef Piece4<D, NV> P;
  static constexpr int NB = (D == 96 ? 128 : D) / (NV ? 16 : 32), QUADS = KEYS / 4, HALF = NB * QUADS;
  static constexpr int W = (2 * HALF + 63) / 64;
  struct Held {
    uint32_t w[W];
  };
  const uint8_t *ks, *vs; // of the head
  uint32_t kst, vst;
  uint32_t off[W];        // of the lane's block and, where a page holds KEYS keys, its first key
  int quad[W];            // that key
  bool v[W];
  bool packed;            // 4 keys of a block are a dword
  uint32_t kfrom[P::SB], vfrom[ALIKE ? 1 : P::SB], kshift, vshift;

  // km, kg, vm, vg: as the lane has its pieces of K and V
  __device__ __forceinline__ Scales4(const Paged4Args &p, int hk, int km, int kg, int vm, int vg) {
    ks = p.ks.s + hk * p.ks.sh, vs = p.vs.s + hk * p.vs.sh;
    kst = (uint32_t)p.ks.st, vst = (uint32_t)p.vs.st, packed = p.packed;
    const int lane = threadIdx.x & 63, blocks = p.a.head_dim / (NV ? 16 : 32);
#pragma unroll
    for (int r = 0; r < W; ++r) {
      const int i = (64 * r + lane) % (2 * HALF), b = i / QUADS % NB;
      v[r] = i >= HALF, quad[r] = 4 * (i % QUADS);
      const uint32_t st = v[r] ? vst : kst, sb = (uint32_t)(v[r] ? p.vs.sb : p.ks.sb);
      off[r] = (b < blocks ? b : 0) * sb + (quad[r] & ((1 << p.a.page_shift) - 1)) * st;
    }
#pragma unroll
    for (int j = 0; j < P::SB; ++j) {
      kfrom[j] = 4 * ((P::block_of(j, kg) * QUADS + km / 4) & 63);
      if constexpr (!ALIKE)
        vfrom[j] = 4 * ((HALF + P::block_of(j, vg) * QUADS + vm / 4) & 63);
    }
    kshift = 8 * (km & 3), vshift = 8 * (vm & 3);
  }
  // Of the keys from n on, a multiple of KEYS.
  template <class Row> __device__ __forceinline__ void load(const Row &pr, int n, Held &x) const {
    const bool one = (1 << pr.shift) >= KEYS; // page
    const uint8_t *bk = ks, *bv = vs;
    if (one) {
      const int e = (n >> pr.shift) - pr.first;
      const uint64_t slot = n & ((1 << pr.shift) - 1);
      bk += pr.template place<1>(e) + slot * kst;
      bv += pr.template place<3>(e) + slot * vst;
    }
#pragma unroll
    for (int r = 0; r < W; ++r) {
      auto step = [&]() { return here_only(v[r] ? vst : kst); };
      if (__builtin_expect(pr.shift >= 2, 1)) { // 4 keys of one page
        const uint8_t *p = (v[r] ? bv : bk) + off[r];
        if (!one) {
          const int e = ((n + quad[r]) >> pr.shift) - pr.first;
          const uint64_t a = pr.template places<1>(e), b = pr.template places<3>(e);
          p += v[r] ? b : a;
        }
        if (__builtin_expect(packed, 1)) {
          x.w[r] = *reinterpret_cast<const uint32_t *>(p);
        } else {
          const uint32_t st = step();
          x.w[r] = (uint32_t)p[0] | (uint32_t)p[st] << 8 | (uint32_t)p[2ull * st] << 16 | (uint32_t)p[3ull * st] << 24;
        }
      } else {
        const int mask = (1 << pr.shift) - 1;
        const uint32_t st = step();
        uint32_t w = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int key = n + quad[r] + t, e = (key >> pr.shift) - pr.first;
          const uint64_t a = pr.template places<1>(e), b = pr.template places<3>(e);
          // (off's part of the quad's first key, whose slot is 0 in pages of 1 and 2)
          w |= (uint32_t)((v[r] ? vs + b : ks + a) + off[r])[(uint64_t)(key & mask) * st] << (8 * t);
        }
        x.w[r] = w;
      }
    }
  }
  // The scale bytes of the lane's pieces of run b.
  template <bool V> __device__ __forceinline__ void of(const Held &x, int b, uint32_t (&s)[P::SB]) const {
#pragma unroll
    for (int j = 0; j < P::SB; ++j) {
      const int r = ((V ? HALF : 0) + P::block_of(j, 0) * QUADS) / 64; // (the other g are in it too)
      const uint32_t at = !V ? kfrom[j] : ALIKE ? kfrom[j] + 4 * (HALF % 64) : vfrom[j % (ALIKE ? 1 : P::SB)];
      const uint32_t w = __builtin_amdgcn_ds_bpermute(at + 16 * b, x.w[r]);
      s[j] = __builtin_amdgcn_ubfe(w, V && !ALIKE ? vshift : kshift, 8);
    }
  }
};

// Q in the type that codes are computed in.  bf16 rows under e4m3 scales become fp16, times the
// power of two that takes the row's largest magnitude to [2^7, 2^8): exact but for what is below
// 2^-31 of that.  Returns what the row's scores are to be multiplied by.  A row with an infinity: its
// scores are infinite or no numbers whatever its other dims are, which have to stay finite.
// x: the lane's dims of a row; the lanes of a row: those that `row_max` goes over.
template <bool BF, int N, class F>
__device__ __forceinline__ float q4_to_f16(u32x4 (&x)[N], F row_max) {
  if constexpr (!BF) {
    return 1.f;
  } else {
    float mx = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mx = fmaxf(mx, fabsf(__uint_as_float((uint32_t)x[c][i] << 16)));
        mx = fmaxf(mx, fabsf(__uint_as_float((uint32_t)x[c][i] & 0xffff0000u)));
      }
    mx = row_max(mx);
    const int e = (__float_as_uint(mx) >> 23) & 255;
    const int up = e == 0 ? 0 : e == 255 ? -120 : 134 - e < 127 ? 134 - e : 127;
    const float f = __builtin_amdgcn_ldexpf(1.f, up);
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const half2_t h = {(_Float16)(__uint_as_float((uint32_t)x[c][i] << 16) * f),
                           (_Float16)(__uint_as_float((uint32_t)x[c][i] & 0xffff0000u) * f)};
        x[c][i] = __builtin_bit_cast(uint32_t, h);
      }
    return e == 255 ? 1.f : __builtin_amdgcn_ldexpf(1.f, -up);
  }
}

// What a row's weights are raised by (PagedFrag::softmax), as an exponent: in fp16 up to 2^15, so that
// a weight loses no more than 2^-32 of the row's sum (without, 2^-25: a row of 131072 small ones 2^-8 of what they
// hold, as much as all of bf16's rounding).
template <bool CBF> constexpr int kUp4 = CBF ? 0 : 7;

// What a unit's beginning and end cost, in steps (paged_sched.h).
constexpr uint32_t kSplit4Overhead = 3, kRows4Overhead = 6;

// Counters of sets of parts begin here in the workspace's 16384 (those of units, and of other
// launches, before them: a launch has at most 768 workgroups).
constexpr uint32_t kSetCounters = 8192;

// Which of 16 keys (four adjacent lanes each) a lane's flag is set of.
__device__ __forceinline__ uint32_t keys_of(uint64_t lanes) {
  uint64_t x = lanes | lanes >> 1;
  x |= x >> 2;
  uint32_t r = 0;
  for (int i = 0; i < 16; ++i)
    r |= (uint32_t)(x >> (4 * i) & 1) << i;
  return r;
}

// ---------------------------------------------------------------------------
// Few rows: the waves of a workgroup share out the keys
// ---------------------------------------------------------------------------

// RT: blocks of 16 rows, which share the fragments of K and V.
template <int D_, bool BF, bool NV_, int RT_> struct Paged4Split {
  static constexpr int D = D_, BN = 32, RT = RT_, ROWS = 16 * RT;
  static constexpr int NS = D == 256 ? 1 : D == 64 ? (RT == 1 ? 6 : 4) : RT == 1 ? 3 : 2; // blocks that a wave has under way
  static constexpr bool NV = NV_, CBF = BF && !NV;
  typedef Code4<CBF, NV> Code;
  typedef PagedFrag16<D, CBF, false, BN> P16; // of the values in 16 bits
  typedef Piece4<D, NV> Piece;
  typedef typename AttnFwd<64, BF, 32, 64>::elt elt; // of q and o
  typedef typename AttnFwd<64, BF, 32, 64>::h4 h4;
  typedef typename P16::h8 h8;
  static constexpr int QUADS = RT * P16::QUADS;
  static constexpr int TILE = P16::TILE, BYTES = TILE > ROWS * D * 4 ? TILE : ROWS * D * 4;
  __device__ __forceinline__ static int quad_at(int row, int qd) {
    return (row >> 4) * P16::QUADS * 64 + P16::quad_at(row & 15, qd);
  }
  // V's tile: 16-byte chunk c of row r lies at c ^ swz(r).  A transposed read takes 32 bytes of each of 8
  // rows: P16's swizzle puts these pairs of chunks on different banks, and bit 0 (which chunk of a pair is
  // first) those that the lanes of 4 keys write together.
  static constexpr int ROW = P16::ROW;
  __device__ __forceinline__ static int swz(int r) { return P16::vswz(r) ^ ((r >> 1) & 1); }
  // V fragments of dim blocks b0 .. b0 + VN - 1 as P16 reads them: the address of the first, from which the
  // others' differ in bits that it has not set.
  static constexpr int VN = D == 256 ? 4 : P16::VN;
  struct Bases {
    uint32_t v[D == 256 ? 1 : P16::NV]; // (heads of 256: 15 registers less; of 128 forming them costs 4%)
  };
  __device__ __forceinline__ static void bases(uint32_t v_lds, Bases &bs) {
    const int lane = threadIdx.x & 63, r = lane & 15, key = 4 * (lane >> 4) + (r >> 2), d = 4 * (r & 3);
    const uint32_t v = v_lds + key * ROW + (((d >> 3) ^ swz(key)) << 4) + (d & 7) * 2;
#pragma unroll
    for (int bd = 0; bd < (D == 256 ? 1 : P16::NV); ++bd)
      bs.v[bd] = v ^ (32 * bd);
  }
  __device__ __forceinline__ static void read_v(const Bases &bs, int b0, i32x4_t (&vf)[VN]) {
    const uint32_t v = here_only(bs.v[0]);
#pragma unroll
    for (int bd = 0; bd < VN; ++bd) {
      const uint32_t a = D == 256 ? v ^ (32 * (b0 + bd)) : bs.v[D == 256 ? 0 : b0 + bd];
      const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)a);
      const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)(a + 16 * P16::ROW));
      vf[bd] = __builtin_bit_cast(i32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// A unit's end: the four waves' sums (quads of 4 dims in smem[wave] by A::quad_at, and each row's
// reference and sum in ms and ls) are joined, and written out, or left as one part of several.
// The last workgroup to arrive joins the parts, in order; where that would be more than one round of
// loads (R parts: 8 a thread, and threads past one set of items take others), the last of each R
// joins those, and the last of all what these leave.  64 parts of 8 rows of 256 dims: a round takes 3
// us, one after the other they took 25.  vs: the scale of v.
template <class A, int BYTES>
__device__ __forceinline__ void paged4_split_end(const PagedAttnArgs &pe, const PagedUnit &ue, float vs,
                                                 uint8_t (&smem)[4][BYTES], float (&ms)[4][A::ROWS],
                                                 float (&ls)[4][A::ROWS], int *flag) {
  constexpr int D = A::D, ROWS = A::ROWS, NJ = 8, kSC1 = 16;
  constexpr int part_bytes = ROWS * (D + 2) * 4;
  typedef typename A::elt elt;
  const int tid = threadIdx.x;
  __syncthreads();
  const int dq = pe.head_dim / 4, items = ue.rows * dq;
  uint8_t *const all = pe.parts;
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(all, 0, 0x7fffffff, 0x00020000);
  // where part j is (a workgroup's two places: paged_sched.h)
  auto part_at = [&](uint32_t j) { return (int)((2 * (ue.w0 + j) + (j == 0 ? ue.slot0 : 0)) * (uint32_t)part_bytes); };
  auto finish = [&](int row, int qd, float mm, float ll, f32x4v x) {
    const int ro = ue.r0 + row;
    const int of = paged_token(pe, ro), h = ue.hk * pe.G + ro - of * pe.G;
    const int64_t t = ue.t0 + of;
    const float f = ll == 0.f ? 0.f : vs / ll;
    typename A::h4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = (elt)(x[e] * f);
    *reinterpret_cast<typename A::h4 *>(static_cast<elt *>(pe.o) + t * pe.o_st + h * pe.o_sh + 4 * qd) = y;
    if (qd == 0 && pe.lse)
      pe.lse[t * pe.Hq + h] = ll == 0.f ? -INFINITY : mm + __builtin_log2f(ll);
  };
  auto store = [&](int at, int row, int qd, float mm, float ll, f32x4v x) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4_t, x), rsrc, at + (row * D + 4 * qd) * 4, 0, kSC1);
    if (qd == 0) {
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(mm), rsrc, at + (ROWS * D + row) * 4, 0, kSC1);
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(ll), rsrc, at + (ROWS * D + ROWS + row) * 4, 0, kSC1);
    }
  };
  for (int it = tid; it < items; it += 256) {
    const int row = it / dq, qd = it % dq;
    float mm = -INFINITY, ll = 0.f;
    f32x4v x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int wv = 0; wv < 4; ++wv)
      paged_join(mm, ll, x, ms[wv][row], ls[wv][row],
                 *reinterpret_cast<const f32x4v *>(smem[wv] + A::quad_at(row, qd) * 16));
    if (ue.parts == 1)
      finish(row, qd, mm, ll, x);
    else
      store(part_at(ue.part), row, qd, mm, ll, x);
  }
  __syncthreads(); // the tiles' and ms' next use
  if (ue.parts == 1)
    return;
  const int groups = items < 256 ? 256 / items : 1;
  // Joins `count` parts, the j-th at from(j).
  auto join = [&](uint32_t count, auto from, auto emit) __attribute__((always_inline)) {
    constexpr int IT = ROWS * D > 1024 ? 2 : 1; // items of a thread at a time
    for (int base = 0; base < items; base += IT * 256) {
      int row[IT], qd[IT];
      bool on[IT];
      float mm[IT], ll[IT];
      f32x4v x[IT];
      const int gi = groups > 1 ? tid / items : 0;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int it = groups > 1 ? tid % items : base + i * 256 + tid;
        on[i] = it < items && gi < groups && (i == 0 || groups == 1);
        row[i] = on[i] ? it / dq : 0, qd[i] = on[i] ? it % dq : 0;
        mm[i] = -INFINITY, ll[i] = 0.f, x[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
      }
      for (uint32_t j0 = gi; j0 < count; j0 += NJ * groups) {
        float pm[IT][NJ], pl[IT][NJ];
        i32x4_t px[IT][NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint32_t jj = j0 + j * groups;
          const int at = from(jj < count ? jj : 0);
#pragma unroll
          for (int i = 0; i < IT; ++i) {
            pm[i][j] = -INFINITY, pl[i][j] = 0.f;
            if (on[i] && jj < count) {
              px[i][j] = __builtin_bit_cast(
                  i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + (row[i] * D + 4 * qd[i]) * 4, 0, kSC1));
              pm[i][j] = __int_as_float(
                  __builtin_amdgcn_raw_buffer_load_b32(rsrc, at + (ROWS * D + row[i]) * 4, 0, kSC1));
              pl[i][j] = __int_as_float(
                  __builtin_amdgcn_raw_buffer_load_b32(rsrc, at + (ROWS * D + ROWS + row[i]) * 4, 0, kSC1));
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < IT; ++i)
            paged_join(mm[i], ll[i], x[i], pm[i][j], pl[i][j], __builtin_bit_cast(f32x4v, px[i][j]));
      }
      if (groups > 1) {
        f32x4v *const xs = reinterpret_cast<f32x4v *>(smem[0]);
        float *const mls = reinterpret_cast<float *>(smem[0] + 4096);
        xs[tid] = x[0];
        mls[tid] = mm[0], mls[256 + tid] = ll[0];
        __syncthreads();
        if (tid < items) {
          for (int k = 1; k < groups; ++k)
            paged_join(mm[0], ll[0], x[0], mls[k * items + tid], mls[256 + k * items + tid], xs[k * items + tid]);
          emit(row[0], qd[0], mm[0], ll[0], x[0]);
        }
        __syncthreads();
      } else {
#pragma unroll
        for (int i = 0; i < IT; ++i)
          if (on[i])
            emit(row[i], qd[i], mm[i], ll[i], x[i]);
      }
    }
  };
  const uint32_t R = NJ * groups;
  if (ue.parts > R) {
    const uint32_t g = ue.part / R, n = ue.parts - g * R < R ? ue.parts - g * R : R, sets = (ue.parts + R - 1) / R;
    // What the parts of set g leave: in the second place of a workgroup whose run lies within the unit,
    // so that it has no other part (the first of the set, of set 0 the second); a last part alone
    // is its set's.  Counters: apart from the units' own, that of the set's first workgroup.
    auto set_at = [&](uint32_t k) {
      return k * R + 1 == ue.parts ? part_at(k * R) : (int)((2 * (ue.w0 + (k ? k * R : 1)) + 1) * (uint32_t)part_bytes);
    };
    if (n > 1) {
      if (!paged_arrive(&pe.counters[kSetCounters + ue.w0 + g * R], n, flag))
        return;
      const int to = set_at(g);
      join(n, [&](uint32_t j) { return part_at(g * R + j); },
           [&](int row, int qd, float mm, float ll, f32x4v x) { store(to, row, qd, mm, ll, x); });
    }
    if (!paged_arrive(&pe.counters[ue.w0], sets, flag))
      return;
    join(sets, set_at, finish);
  } else {
    if (!paged_arrive(&pe.counters[ue.w0], ue.parts, flag))
      return;
    join(ue.parts, part_at, finish);
  }
}

// f(0), .. f(N - 1), of constants.
template <int N, class F, int... I>
__device__ __forceinline__ void each_slot(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F> __device__ __forceinline__ void each_slot(F f) {
  each_slot<N>(f, std::make_integer_sequence<int, N>());
}

// Workgroups of a CU: by LDS, and by registers where heads are long.
template <class A> constexpr int paged4_split_groups() { return A::BYTES * 4 <= 81920 ? 2 : 1; }

// A wave takes a quarter of a unit's blocks of 32 keys, one after the other and by itself, NS blocks of codes
// under way: codes, scales and page numbers are in registers before they are needed, and no barrier stands
// between a unit's begin and its end.  Bound by how many bytes are under way.  One token for each of 32 sequences of 100 .. 16384
// keys, 32 heads of 128 over 8: 36.5 us, 3.3 TB/s (33 us with the arithmetic taken out); 4 tokens for each of 4
// sequences of 60000 .. 131072: 101 us, 4.5 TB/s (94); 8 sequences of 5000 .. 32768, 16 heads of 256 over 2, one
// block under way for lack of registers: 35 us, 2.0 TB/s (31).  One token over 1500 keys: 10 us, of which the
// launch, the table, the codes behind it and the join of the parts each wait for memory once.
template <class A>
__global__ void __launch_bounds__(256, paged4_split_groups<A>()) paged_attn4_split_kernel(Paged4Args args4) {
  constexpr int D = A::D, BN = A::BN, RT = A::RT, ROWS = A::ROWS, NS = A::NS;
  typedef typename A::P16 P16;
  typedef typename A::Piece Piece;
  typedef typename A::Code Code;
  typedef typename A::elt elt;
  typedef PagedSched<ROWS, BN, 4, kSplit4Overhead> Sched;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4][A::BYTES];
  __shared__ float ms[4][ROWS], ls[4][ROWS];
  __shared__ PagedSchedState st;
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  if (wave == 0) {
    Sched sched(args4.a, st);
    sched.init(blockIdx.x, gridDim.x);
    sched.get(st.unit[0]);
  }
  __syncthreads();

  const uint32_t v_lds = lds_addr(smem[wave]);
  typename A::Bases bs;
  A::bases(v_lds, bs);
  const int km = lane & 15, kg = lane >> 4, vm = lane >> 2, vg = lane & 3;
  // where the lane's first 8 dims of V go in the tile (16 rows on: 16 * ROW; dword c: at ^ Piece::at(c))
  const uint32_t vw = v_lds + vm * P16::ROW + (((Piece::dim(0, vg) / 8) ^ A::swz(vm)) << 4);

  for (int turn = 0;; turn ^= 1) {
    const Paged4Args &p4 = paged4_args();
    const PagedAttnArgs &p = p4.a;
    const PagedUnit un = paged_unit(st.unit[turn]);
    if (un.rows <= 0)
      break;
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
    PageRow4<true> pr{{p.table + un.b * p.table_s, (uint32_t)p.table_width, p.pages, p.page_shift}, {}};
    const Side4<D, A::NV, false> sk(p4, un.hk, km, kg);
    const Side4<D, A::NV, true> sv(p4, un.hk, vm, vg);
    // The table, Q and the first blocks are under way together, and meanwhile the first wave
    // looks up the next unit.
    if (k0 < k1)
      pr.load(k0 * BN);
    u32x4 qf[RT][Piece::KW];
    int rr[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = 16 * i + km;
      rr[i] = un.r0 + (r < un.rows ? r : 0);
      const int of = paged_token(p, rr[i]), head = un.hk * p.G + rr[i] - of * p.G;
      const elt *row = static_cast<const elt *>(p.q) + (int64_t)(un.t0 + of) * p.q_st + head * p.q_sh;
#pragma unroll
      for (int c = 0; c < Piece::KW; ++c) {
        const int d = Piece::dim(c, kg);
        qf[i][c] = *reinterpret_cast<const u32x4 *>(row + (d < p.head_dim ? d : 0));
      }
    }
    const Scales4<D, A::NV, BN, false> sc(p4, un.hk, km, kg, vm, vg);
    Piece kp[NS][2], vp[NS][2];
    typename Scales4<D, A::NV, BN, false>::Held sp[NS];
    uint32_t here[NS + 1] = {}; // of blocks k .. k + NS
    if (k0 < k1) {
      pr.settle();
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (k0 + i < k1) {
          const int n = (k0 + i) * BN;
          pr.hold(n);
          here[i] = (uint32_t)pr.template there<BN>(n, un.hi);
          sc.load(pr, n, sp[i]);
          sk.template load<true>(pr, n, km, kp[i]), sv.template load<true>(pr, n, vm, vp[i]);
        }
    }
    if (wave == 0)
      Sched(p, st).get(st.unit[turn ^ 1]);
    int lo[RT], hi[RT]; // of the lane's rows
#pragma unroll
    for (int i = 0; i < RT; ++i)
      paged_keys(p, un.pos0, un.len, rr[i], rr[i] + 1, lo[i], hi[i]);
    // keys that every row attends to
    int lo_all, hi_all, skip;
    paged_keys(p, un.pos0, un.len, un.r0, un.r0 + 1, skip, hi_all);
    paged_keys(p, un.pos0, un.len, un.r0 + un.rows - 1, un.r0 + un.rows, lo_all, skip);
    const float scale0 = p.qk_scale * (p.k_scale ? p.k_scale[un.hk] : 1.f);
    float scale[RT]; // of the lane's rows
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const bool live = 16 * i + km < un.rows;
#pragma unroll
      for (int c = 0; c < Piece::KW; ++c)
        qf[i][c] = __builtin_bit_cast(
            u32x4, P16::P32::settled(__builtin_bit_cast(typename P16::h8, qf[i][c]),
                                     live && Piece::dim(c, kg) < p.head_dim, scale0));
      scale[i] = scale0 == 0.f ? 1.f : fabsf(scale0);
      if constexpr (A::NV)
        scale[i] *= q4_to_f16<!std::is_same<elt, _Float16>::value>(
            qf[i], [](float v) { return P16::row_max(v); });
    }
    float m[RT], l[RT];
    typename P16::Acc acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
      for (int b = 0; b < P16::NV; ++b)
        acc[i][b] = typename P16::f4v{};
    }
    auto iter = [&](int k, auto slot_c) __attribute__((always_inline)) {
      constexpr int SL = decltype(slot_c)::value;
      const int n0 = k * BN, na = n0 + NS * BN;
      typename P16::Scores s[RT];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const Piece &x = kp[SL][b];
        uint32_t f[Piece::SB];
        sc.template of<false>(sp[SL], b, f);
#pragma unroll
        for (int j = 0; j < Piece::SB; ++j)
          f[j] = Code::factor(f[j], false);
#pragma unroll
        for (int i = 0; i < RT; ++i)
          s[i][b] = typename P16::f4v{};
#pragma unroll
        for (int c = 0; c < Piece::KW; ++c) {
          const auto kf = __builtin_bit_cast(typename P16::h8, Code::eight(x.w[c], f[Piece::scale_of(c)]));
#pragma unroll
          for (int i = 0; i < RT; ++i)
            s[i][b] = P16::mfma(kf, __builtin_bit_cast(typename P16::h8, qf[i][c]), s[i][b]);
        }
      }
      const uint32_t vto = here_only(vw);
      uint64_t none[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const Piece &x = vp[SL][b];
        uint32_t f[Piece::SB];
        sc.template of<true>(sp[SL], b, f);
        bool bad = false;
#pragma unroll
        for (int j = 0; j < Piece::SB; ++j)
          bad = bad || Code::bad(f[j]), f[j] = Code::factor(f[j], true);
        none[b] = __ballot(bad);
#pragma unroll
        for (int c = 0; c < Piece::KW; ++c) {
          typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
          *(lds_u32x4 *)(uintptr_t)((vto ^ Piece::at(c)) + b * 16 * P16::ROW) = Code::eight(x.w[c], f[Piece::scale_of(c)]);
        }
      }
      if (k + NS < k1) {
        pr.hold(na);
        here[NS] = (uint32_t)pr.template there<BN>(na, un.hi);
        sc.load(pr, na, sp[SL]);
        sk.template load<true>(pr, na, km, kp[SL]), sv.template load<true>(pr, na, vm, vp[SL]);
      }
      if (__builtin_expect((none[0] | none[1]) != 0, 0)) {
        const uint32_t nan = (keys_of(none[0]) | keys_of(none[1]) << 16) >> (4 * kg);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[i][b][r] = nan >> (16 * b + r) & 1 ? __builtin_nanf("") : s[i][b][r];
      }
      typename P16::PF pf[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (here[0] != ~0u || n0 < lo_all || n0 + BN > hi_all) {
          const int a = lo[i] - n0 < 0 ? 0 : lo[i] - n0, z = hi[i] - n0 < 0 ? 0 : hi[i] - n0;
          uint64_t seen = z < 64 ? (1ull << z) - 1 : ~0ull;
          seen &= a < 64 ? ~0ull << a : 0;
          P16::mask(s[i], seen & here[0]);
        }
        P16::template softmax<kUp4<A::CBF>>(s[i], scale[i], acc[i], m[i], l[i], pf[i]);
      }
#pragma unroll
      for (int b0 = 0; b0 < P16::NV; b0 += A::VN) {
        i32x4_t vf[A::VN];
        A::read_v(bs, b0, vf);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int bd = 0; bd < A::VN; ++bd)
            acc[i][b0 + bd] = P16::mfma(__builtin_bit_cast(typename P16::h8, vf[bd]), pf[i][0], acc[i][b0 + bd]);
      }
#pragma unroll
      for (int i = 0; i < NS; ++i)
        here[i] = here[i + 1];
    };
    for (int k = k0; k < k1;)
      each_slot<NS>([&](auto slot) __attribute__((always_inline)) {
        if (k < k1)
          iter(k++, slot);
      });

    // The waves' sums: quads of 4 dims in lane order in each one's own tile.
    const PagedAttnArgs &pe = paged_args();
    const PagedUnit ue = paged_unit(st.unit[turn]);
    const float vs = pe.v_scale ? pe.v_scale[ue.hk] : 1.f;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      l[i] = P16::row_sum(l[i]);
      if (k0 < k1) {
#pragma unroll
        for (int q = 0; q < P16::QUADS; ++q)
          *reinterpret_cast<f32x4v *>(smem[wave] + ((i * P16::QUADS + q) * 64 + lane) * 16) =
              P16::quad(acc[i], q);
      }
      if (lane < 16)
        ms[wave][16 * i + lane] = m[i], ls[wave][16 * i + lane] = l[i];
    }
    paged4_split_end<A>(pe, ue, vs, smem, ms, ls, &flag);
  }
  paged_zero_rows<elt>(args4.a);
}

// ---------------------------------------------------------------------------
// Many rows: the waves of a workgroup share the keys
// ---------------------------------------------------------------------------

// 128 rows a unit, 32 a wave.  Of a block of 64 keys each wave holds the codes of 16, converts them
// into the tiles of 16-bit rows that all four read, and loads those of the next block: K and V have
// two tiles each, one barrier a block.  (K goes through LDS here: each wave alone would convert it
// four times.)
//
// Bound by the work between the products: a block's conversions, exponentials, masks and LDS accesses
// take about as long as its MFMAs, and two workgroups a CU (heads of 64: three), which is what registers
// allow, overlap only part of them.  2 sequences of 2048 new tokens over up to 16384 keys, 32 heads of 128
// over 8: 1052 us, 0.84 PFLOP/s of the 1.26 that a large product of the library reaches (1102 before
// V's tile had its swizzle; the 16-bit cache's form, which converts nothing, takes 970).  24 sequences of 1 ..
// 300 tokens, 16 heads of 64, window 1024: 42 us with a head's tokens together, 48 to 50 with a token's heads
// together, where four heads share a line that each workgroup fetches by itself.
template <int D_, bool BF, bool NV_> struct Paged4Rows {
  static constexpr int D = D_, BN = 64;
  static constexpr bool NV = NV_, CBF = BF && !NV;
  typedef Code4<CBF, NV> Code;
  typedef PagedFrag<D, CBF, false, BN> P;
  typedef Piece4<D, NV> Piece;
  typedef typename AttnFwd<64, BF, 32, 64>::elt elt; // of q and o
  // V's tile: P's swizzle puts the 64 bytes of 4 rows that a transposed read takes on different banks, and
  // the same bits again those within 64 that the lanes of 4 keys write together (without: a quarter of
  // the LDS's time).
  __device__ __forceinline__ static int swz(int r) { return 5 * (P::vswz(r) / 4); }
  // Fragments as P reads them, from one address each of K and V: those of the other chunks and dim blocks
  // differ in bits that the first has not set.
  __device__ __forceinline__ static uint32_t v_base(uint32_t v_lds) {
    const int lane = threadIdx.x & 63, L = lane & 15, key = 4 * (lane >> 5) + (L >> 2);
    const int d = 16 * ((lane >> 4) & 1) + 4 * (L & 3);
    return v_lds + key * P::ROW + (((d >> 3) ^ swz(key)) << 4) + (d & 7) * 2;
  }
  __device__ __forceinline__ static void read_k(uint32_t k, int at, typename P::KF &kf) {
    typedef __attribute__((address_space(3))) i32x4_t lds_i32x4;
#pragma unroll
    for (int c = 0; c < P::NK; ++c)
#pragma unroll
      for (int b = 0; b < BN / 32; ++b)
        kf.v[b][c] = *(const lds_i32x4 *)(uintptr_t)((k ^ (32 * c)) + at + b * 32 * P::ROW);
  }
  template <int N>
  __device__ __forceinline__ static void read_v(uint32_t v, int at, int b0, typename P::template VF<N> &vf) {
#pragma unroll
    for (int bd = 0; bd < N; ++bd)
#pragma unroll
      for (int c = 0; c < BN / 16; ++c) {
        const uint32_t a = (v ^ (64 * (b0 + bd))) + at + c * 16 * P::ROW;
        const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)a);
        const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(uintptr_t)(a + 8 * P::ROW));
        vf.v[bd][c] = __builtin_bit_cast(i32x4_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
  }
  static constexpr int VR = D <= 128 ? P::NV : P::VN; // dim blocks of V read ahead of the softmax
};

// A unit's end: its rows (32 a wave) are written out as T, or left as one part of several, which the
// last workgroup to arrive joins, in order; of more than kRowsSet parts in sets, as
// paged4_split_end.  460 rows of one sequence (heads of 128) over 14470 keys: 42 us, 97 part by part.
constexpr uint32_t kRowsSet = 8;
template <class P, class T>
__device__ __forceinline__ void paged4_rows_end(const PagedUnit &unit, typename P::Acc &acc, float m, float l,
                                                int *flag) {
  constexpr int D = P::D, kSC1 = 16;
  constexpr int64_t part_bytes = 128 * (D + 2) * 4;
  typedef T T4 __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  l = P::X::xsum(l);
  const PagedAttnArgs &pe = paged_args();
  const PagedUnit ue = paged_unit(unit);
  __syncthreads(); // (the first wave will write the unit after the next there)
  const float vs = pe.v_scale ? pe.v_scale[ue.hk] : 1.f;
  const int r = 32 * wave + (lane & 31), rr = ue.r0 + (r < ue.rows ? r : 0);
  const bool busy = ue.rows > 32 * wave;
  if (ue.parts > 1) {
    auto place = [&](uint64_t slot) {
      return __builtin_amdgcn_make_buffer_rsrc(pe.parts + slot * part_bytes, 0, (int)part_bytes, 0x00020000);
    };
    auto part_at = [&](uint32_t j) -> uint64_t { return 2ull * (ue.w0 + j) + (j == 0 ? ue.slot0 : 0); };
    // (lane order: quads of a wave side by side)
    auto store = [&](uint64_t slot) __attribute__((always_inline)) {
      if (!busy)
        return;
      const auto to = place(slot);
#pragma unroll
      for (int q = 0; q < D / 8; ++q)
        __builtin_amdgcn_raw_buffer_store_b128(
            __builtin_bit_cast(i32x4_t, f32x4v{acc[q / 4][4 * (q % 4)], acc[q / 4][4 * (q % 4) + 1],
                                               acc[q / 4][4 * (q % 4) + 2], acc[q / 4][4 * (q % 4) + 3]}),
            to, ((wave * (D / 8) + q) * 64 + lane) * 16, 0, kSC1);
      if (g == 0) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(m), to, (128 * D + r) * 4, 0, kSC1);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(l), to, (128 * D + 128 + r) * 4, 0, kSC1);
      }
    };
    constexpr uint32_t R = kRowsSet;
    // (places and counters of sets: as in paged4_split_end)
    const uint32_t s = ue.part / R, sets = (ue.parts + R - 1) / R;
    auto set_at = [&](uint32_t k) -> uint64_t {
      return k * R + 1 == ue.parts ? part_at(k * R) : 2ull * (ue.w0 + (k ? k * R : 1)) + 1;
    };
    bool last = ue.parts <= R; // what is joined next is all of the unit, not a set
    uint32_t n = last ? ue.parts : ue.parts - s * R < R ? ue.parts - s * R : R;
    uint64_t to = part_at(ue.part);
    if (n == 1) // a set of one part: that is what it leaves
      last = true, n = sets;
    for (;; last = true, n = sets, to = set_at(s)) {
      store(to);
      if (!paged_arrive(&pe.counters[last ? ue.w0 : kSetCounters + ue.w0 + s * R], n, flag))
        return;
      if (busy) {
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (int bd = 0; bd < D / 32; ++bd)
          acc[bd] = typename P::f16v{};
#pragma nounroll
        for (uint32_t j = 0; j < n; ++j) {
          const auto part = place(!last ? part_at(s * R + j) : ue.parts <= R ? part_at(j) : set_at(j));
          i32x4_t x[D / 8];
#pragma unroll
          for (int q = 0; q < D / 8; ++q)
            x[q] = __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                                   part, ((wave * (D / 8) + q) * 64 + lane) * 16, 0, kSC1));
          const float m1 = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(part, (128 * D + r) * 4, 0, kSC1));
          const float l1 = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(part, (128 * D + 128 + r) * 4, 0, kSC1));
          if (l1 == 0.f) // nothing (a NaN among the scores makes it NaN)
            continue;
          const float up = fmaxf(m, m1);
          const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - up);
          const float a1 = __builtin_amdgcn_exp2f(m1 - up);
          l = l * a + l1 * a1;
          m = up;
#pragma unroll
          for (int q = 0; q < D / 8; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[q / 4][4 * (q % 4) + e] = acc[q / 4][4 * (q % 4) + e] * a + __int_as_float(x[q][e]) * a1;
        }
      }
      if (last)
        break;
    }
  }
  if (r < ue.rows) {
    const int of = paged_token(pe, rr), head = ue.hk * pe.G + rr - of * pe.G;
    const int64_t tok = ue.t0 + of;
    const float f = l == 0.f ? 0.f : vs / l;
    T *const orow = static_cast<T *>(pe.o) + tok * pe.o_st + head * pe.o_sh;
#pragma unroll
    for (int q = 0; q < D / 8; ++q) {
      const int d = 32 * (q / 4) + 8 * (q % 4) + 4 * g;
      T4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = (T)(acc[q / 4][4 * (q % 4) + e] * f);
      if (d < pe.head_dim)
        *reinterpret_cast<T4 *>(orow + d) = y;
    }
    if (g == 0 && pe.lse)
      pe.lse[tok * pe.Hq + head] = l == 0.f ? -INFINITY : m + __builtin_log2f(l);
  }
}

template <class A> constexpr int paged4_rows_groups() { return A::D > 128 ? 1 : A::D > 64 ? 2 : 3; }

template <class A>
__global__ void __launch_bounds__(256, paged4_rows_groups<A>()) paged_attn4_rows_kernel(Paged4Args args4) {
  constexpr int D = A::D, BN = A::BN;
  typedef typename A::P P;
  typedef typename A::Piece Piece;
  typedef typename A::Code Code;
  typedef typename A::elt elt;
  typedef PagedSched<128, BN, 1, kRows4Overhead> Sched;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * P::TILE];
  __shared__ PagedSchedState st;
  __shared__ uint32_t nans[2][4]; // of each wave's 16 keys of a tile, those without numbers in V
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  if (wave == 0) {
    Sched sched(args4.a, st);
    const uint32_t n = gridDim.x, b = blockIdx.x; // (XCDs: as in paged_attn_rows_kernel)
    sched.init(n % 8 == 0 ? (b % 8) * (n / 8) + b / 8 : b, n);
    sched.get(st.unit[0]);
  }
  __syncthreads();

  const uint32_t k_lds = lds_addr(smem), v_lds = k_lds + 2 * P::TILE;
  typename P::Bases bs;
  P::bases(k_lds, v_lds, bs);
  bs.v[0] = A::v_base(v_lds);
  const int em = lane >> 2, eg = lane & 3, er = 16 * wave + em; // the key of a block that the lane converts
  const uint32_t kw = k_lds + er * P::ROW + (((Piece::dim(0, eg) / 8) ^ P::kswz(er)) << 4);
  const uint32_t vw = v_lds + er * P::ROW + (((Piece::dim(0, eg) / 8) ^ A::swz(er)) << 4);

  for (int turn = 0;; turn ^= 1) {
    const Paged4Args &p4 = paged4_args();
    const PagedAttnArgs &p = p4.a;
    const PagedUnit un = paged_unit(st.unit[turn]);
    if (un.rows <= 0)
      break;
    int k0 = 0, k1 = 0;
    if (un.hi > un.lo) {
      const int first = un.lo / BN, last = (int)(((int64_t)un.hi + BN - 1) / BN);
      k0 = first + (int)un.s0;
      k1 = first + (int)un.s1 < last ? first + (int)un.s1 : last;
    }
    PageRow4<false> pr{{p.table + un.b * p.table_s, (uint32_t)p.table_width, p.pages, p.page_shift}, {}};
    const Side4<D, A::NV, false> sk(p4, un.hk, em, eg);
    const Side4<D, A::NV, true> sv(p4, un.hk, em, eg);
    uint64_t here[3] = {}; // of blocks k, k + 1, k + 2
    const Scales4<D, A::NV, 16, true> sc(p4, un.hk, em, eg, em, eg);
    struct Codes { // of 16 keys
      Piece k[1], v[1];
      typename Scales4<D, A::NV, 16, true>::Held s;
    } next;
    const bool once = un.alone; // keys that no other unit reads go past the caches
    auto fetch = [&](int k, Codes &x) __attribute__((always_inline)) {
      pr.hold(k * BN);
      here[2] = pr.template there<BN>(k * BN, un.hi);
      const int n = k * BN + 16 * wave;
      sc.load(pr, n, x.s);
      if (once)
        sk.template load<true>(pr, n, em, x.k), sv.template load<true>(pr, n, em, x.v);
      else
        sk.template load<false>(pr, n, em, x.k), sv.template load<false>(pr, n, em, x.v);
    };
    auto convert = [&](int slot, const Codes &x) __attribute__((always_inline)) {
      typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
      uint32_t fk[Piece::SB], fv[Piece::SB];
      sc.template of<false>(x.s, 0, fk), sc.template of<true>(x.s, 0, fv);
      bool bad = false;
#pragma unroll
      for (int j = 0; j < Piece::SB; ++j) {
        bad = bad || Code::bad(fv[j]);
        fk[j] = Code::factor(fk[j], false), fv[j] = Code::factor(fv[j], true);
      }
      const uint32_t kto = here_only(kw), vto = here_only(vw);
      const uint64_t none = __ballot(bad);
      if (lane == 0)
        nans[slot][wave] = none ? keys_of(none) : 0;
#pragma unroll
      for (int c = 0; c < Piece::KW; ++c) {
        *(lds_u32x4 *)(uintptr_t)((kto ^ Piece::at(c)) + slot * P::TILE) = Code::eight(x.k[0].w[c], fk[Piece::scale_of(c)]);
        *(lds_u32x4 *)(uintptr_t)((vto ^ Piece::at(c)) + slot * P::TILE) = Code::eight(x.v[0].w[c], fv[Piece::scale_of(c)]);
      }
    };
    // The table, Q and the first blocks are under way together, and meanwhile the first wave
    // looks up the next unit.
    if (k0 < k1)
      pr.load(k0 * BN);
    const bool busy = un.rows > 32 * wave;
    const int r = 32 * wave + (lane & 31), rr = un.r0 + (r < un.rows ? r : 0);
    const int of = paged_token(p, rr), head = un.hk * p.G + rr - of * p.G;
    const elt *qrow = static_cast<const elt *>(p.q) + (int64_t)(un.t0 + of) * p.q_st + head * p.q_sh;
    u32x4 qx[D / 16];
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const int d = P::q_dim(c);
      qx[c] = *reinterpret_cast<const u32x4 *>(qrow + (d < p.head_dim ? d : 0));
    }
    // (two blocks' codes at once where there are registers for them)
    constexpr bool BOTH = D <= 64;
    Codes other;
    Codes &begin = BOTH ? other : next;
    auto second = [&]() __attribute__((always_inline)) {
      if (k0 + 1 < k1) {
        fetch(k0 + 1, next);
        here[1] = here[2];
      }
    };
    if (k0 < k1) {
      pr.settle();
      fetch(k0, begin);
      here[0] = here[2];
      if constexpr (BOTH)
        second();
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
    const float scale0 = p.qk_scale * (p.k_scale ? p.k_scale[un.hk] : 1.f);
    typename P::QF qf;
    float scale = scale0 == 0.f ? 1.f : fabsf(scale0);
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      qx[c] = __builtin_bit_cast(u32x4, P::settled(__builtin_bit_cast(typename P::h8, qx[c]),
                                                   r < un.rows && P::q_dim(c) < p.head_dim, scale0));
    if constexpr (A::NV)
      scale *= q4_to_f16<!std::is_same<elt, _Float16>::value>(qx, [](float v) { return P::X::xmax(v); });
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      qf.v[c] = __builtin_bit_cast(typename P::h8, qx[c]);
    float m = -INFINITY, l = 0.f;
    typename P::Acc acc = {};
    typename P::Scores s;
    if (k0 < k1) {
      convert(0, begin);
      if constexpr (!BOTH)
        second();
    }
    __syncthreads();
    auto iter = [&](int k, auto slot_c) __attribute__((always_inline)) {
      constexpr int SL = decltype(slot_c)::value;
      const int n0 = k * BN;
      const bool on = live(k);
      if (k + 1 < k1)
        convert(1 - SL, next);
      if (on) {
        typename P::KF kf;
        A::read_k(here_only(bs.k[0]), SL * P::TILE, kf);
        if constexpr (D <= 128)
          __builtin_amdgcn_sched_barrier(0);
        P::qk(kf, qf, s);
      }
      __builtin_amdgcn_sched_barrier(0); // (the codes' registers are K's fragments' before)
      if (k + 2 < k1)
        fetch(k + 2, next);
      if (on) {
        constexpr int VR = A::VR;
        typename P::template VF<VR> vf;
        A::read_v(here_only(bs.v[0]), SL * P::TILE, 0, vf);
        __builtin_amdgcn_sched_barrier(0);
        uint64_t nan = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          nan |= (uint64_t)(uint32_t)uniform((int)nans[SL][w]) << (16 * w);
        if (__builtin_expect(nan != 0, 0)) {
          nan >>= 4 * g;
#pragma unroll
          for (int b = 0; b < BN / 32; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              s[b][e] = nan >> (32 * b + 8 * (e / 4) + e % 4) & 1 ? __builtin_nanf("") : s[b][e];
        }
        if (here[0] != ~0ull || n0 < lo_all || n0 + BN > hi_all) {
          const int a = lo - n0 < 0 ? 0 : lo - n0, z = hi - n0 < 0 ? 0 : hi - n0;
          uint64_t seen = z < 64 ? (1ull << z) - 1 : ~0ull;
          seen &= a < 64 ? ~0ull << a : 0;
          P::mask(s, seen & here[0]);
        }
        typename P::PF pf;
        P::template softmax<kUp4<A::CBF>>(s, scale, acc, m, l, pf);
        P::pv(vf, 0, pf, acc);
#pragma unroll
        for (int b0 = VR; b0 < P::NV; b0 += VR) {
          A::read_v(here_only(bs.v[0]), SL * P::TILE, b0, vf);
          P::pv(vf, b0, pf, acc);
        }
      }
      here[0] = here[1], here[1] = here[2];
      __syncthreads();
    };
    for (int k = k0; k < k1;) {
      iter(k++, std::integral_constant<int, 0>());
      if (k < k1)
        iter(k++, std::integral_constant<int, 1>());
    }
    paged4_rows_end<P, elt>(st.unit[turn], acc, m, l, &flag);
  }
  paged_zero_rows<elt>(args4.a);
}

} // namespace txk
