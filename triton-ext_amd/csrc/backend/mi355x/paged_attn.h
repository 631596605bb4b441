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

#include "paged_frag.h"
#include "rotary.h"

namespace txk {

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
// blocks, with LDS tiles of its own that are loaded again as soon as their fragments are in
// registers, and no barrier; at the end the four join in LDS.  Bound by memory: 8 waves a CU
// keep up to 16 KiB each in flight, and what a block computes (half as much on 16 rows) hides
// behind the other waves' loads.  One token of each of 32 sequences of 145 .. 16384, 32 heads of
// 128 over 8: 86 us, 5.3 TB/s (the same on 32 rows a unit: 90; loads that are kept in the caches:
// 100); four drafted tokens of each of 4 sequences of up to 131072 in e4m3: 158 us, 5.1 TB/s (one
// tile of 64 keys in place of two of 32: 179).  A call of few keys is the chain of its phases: lengths,
// table, keys, the join of the parts: one sequence of 1500, 9.8 us, of which the loop 1.
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
    sched.init(blockIdx.x, gridDim.x);
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
    auto iter = [&](int k, auto slot_c) __attribute__((always_inline)) {
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
// of K's fragments are under way before the first of their MFMAs, all of V's before the softmax.
// Bound by the matrix cores and the softmax's VALU work in turn: chunks of 2048 tokens of two
// sequences of 11869 and 16384 keys, 32 heads of 128 over 8: 970 us (960 .. 980 from card to card),
// 907 TFLOP/s, the MFMAs busy 51% of the time, the VALU 46%, at 1.7 GHz under the power limit (S_{k+1}
// computed beside the softmax of S_k, which leaves registers for single fragments: 1% more; s_setprio
// around the MFMAs: 5% more).  24
// sequences of 1 .. 300 tokens with a window, heads of 64: 36 us, bound by the beginning and end of
// units (about 7 us each).
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
    // the 8 XCDs take contiguous runs: a head's keys stay in one L2 (chunks of 2048: 2% less)
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
    // Keys that no other unit reads go past the caches (64 rows of each of 16 sequences of 16384 keys:
    // 230 -> 209 us); those that others do must not (chunks of 2048: 20% more).
    const bool once = un.alone;
    auto issue = [&](const PageSide &sd, int k, const uint32_t (&off)[U],
                     uint32_t lds) __attribute__((always_inline)) {
      if (once)
        issue_rows<A, U, true>(pr, sd, k * BN, un.hi, U * wave, off, lds, row_bytes);
      else
        issue_rows<A, U, false>(pr, sd, k * BN, un.hi, U * wave, off, lds, row_bytes);
    };
    auto issue_k = [&](int k, int slot) __attribute__((always_inline)) { issue(sk, k, ko, k_lds + slot * A::TILE); };
    auto issue_v = [&](int k, int slot) __attribute__((always_inline)) { issue(sv, k, vo, v_lds + slot * A::TILE); };
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
    auto iter = [&](int k, auto slot_c) __attribute__((always_inline)) {
      constexpr int SL = decltype(slot_c)::value;
      const int n0 = k * BN;
      const bool on = live(k);
      if (k + 1 < k1)
        issue_v(k + 1, 1 - SL);
      if (on) {
        typename A::KF kf;
        A::read_k(bs, SL * A::TILE, kf);
        if constexpr (D <= 128)
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
        constexpr int VR = D <= 128 ? A::NV : A::VN; // dim blocks read ahead (256 dims: for want of registers)
        typename A::template VF<VR> vf;
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
#pragma unroll
        for (int b0 = VR; b0 < A::NV; b0 += VR) {
          A::read_v(bs, SL * A::TILE, b0, vf);
          A::pv(vf, b0, pf, acc);
        }
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
