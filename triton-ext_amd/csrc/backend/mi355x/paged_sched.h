// Which workgroup of a paged attention launch does what (paged_attn.h): its arguments, the units of
// work, how they are dealt out, and how parts of one are joined.
#pragma once

#include <hip/hip_runtime.h>

#include "decode_i8.h"
#include "gemm16_w4.h"

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
  uint32_t pages;
  uint32_t g_mul, g_shift; // n / G = mulhi(n, g_mul) >> g_shift for n < 2^31 (G 1: g_mul 0)
  int32_t most; // keys that a table row has place for
  int32_t T, B, G, Hq, Hkv, head_dim, page_shift, causal, window;
  int32_t k_run, v_run; // rows of one resource
  float qk_scale;       // sm_scale / ln 2
};

__device__ __forceinline__ int lane_value(int v, int lane) {
  return __builtin_amdgcn_readlane(v, lane);
}
__device__ __forceinline__ int64_t lane_value64(int64_t v, int lane) {
  return (int64_t)(uint32_t)lane_value((int)v, lane) | (int64_t)lane_value((int)(v >> 32), lane) << 32;
}
// A unit of work: rows r0 .. r0 + rows - 1 of sequence b and kv head hk, whose tokens begin at
// row t0 of q and at position pos0, and of its steps those from s0 to s1.  Cut in parts,
// this one is `part`; part j is that of workgroup w0 + j, in its first place of the workspace, but
// part 0 in place slot0 (a workgroup's run has a cut unit at its beginning or at its end).
struct alignas(16) PagedUnit {
  int64_t pos0;
  int t0, r0, rows, hk, b, len, lo, hi; // keys [lo, hi)
  uint32_t s0, s1, parts, part, w0, slot0 : 1, alone : 1; // alone: the sequence's only unit of hk
};
static_assert(sizeof(PagedUnit) == 64, "four 16-byte reads");

// What a unit's beginning and end cost, in steps.  32 sequences of 145 .. 16384 tokens (17 of them
// under 2000): 100 us with 2 and the next unit looked up under the first loads, 124 without either;
// mixed lengths with a window: 37.9 with 4, 36.3 with 6, 37.1 with 9.
constexpr uint32_t kSplitOverhead = 2, kRowsOverhead = 6;

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
// begins with OV more that stand for what its beginning and end cost.  The first wave goes through
// this, a lane per sequence (64 at a time, in LDS) or block of rows; sums across lanes.
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
    const uint32_t share = total > grid ? (total + grid - 1) / grid : 1;
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
        u.parts = 1, u.part = 0, u.w0 = 0, u.slot0 = 0, u.alone = rows == nr;
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
  u.parts = v[3][0], u.part = v[3][1], u.w0 = v[3][2], u.slot0 = v[3][3] & 1, u.alone = v[3][3] >> 1 & 1;
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

} // namespace txk
