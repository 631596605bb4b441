// The books of a paged cache (page table, lengths, reference counts) and the moves
// of its pages.
//
// The books are integers: what bounds these kernels is the chain of their phases, not the bytes.
// So a launch has as many workgroups as the table's rows fill, and every one works out
// by itself what it needs of the others' part (sums over the sequences, which pages
// are free), rather than wait for it.  That needs the books that all read to stay as they are:
// where counts or lengths are written in place, the launch has one workgroup.  Free pages are
// taken in ascending order whatever the timing, so results do not depend on it.
// 256 rows of 512 entries and 65536 pages: page_reserve 6.5 us (one workgroup: 129) where
// free pages lie at the front, 34 a call where they come after 65000 that are held; 64 rows of 256
// and 4096 pages: page_compact's books 9.3 us (19.6), page_free 4.7 and the counts' copy 2.2 (19.6);
// 56 children of 64 entries: page_fork's 8.6 us (11).
// Pages are copied by a kernel of their own that takes its list (and, compacting, its
// length) from device memory.
#pragma once

#include <hip/hip_runtime.h>

#include "tile_common.h"
#include "triton_ext/tx_cache.h"

namespace txk {

constexpr int kBookThreads = 512, kBookWaves = kBookThreads / 64;
constexpr int kBookRows = 512; // rows of the table that a workgroup takes at a time

struct BookArgs {
  int64_t W;
  int32_t S, P, n, page_shift;
  int32_t rows;              // rows of a workgroup, at most kBookRows
  int32_t table_in_place, refs_in_place;
  const int32_t *table, *len, *refs;
  const int32_t *new_len, *parent, *child;
  const uint8_t *drop;
  int32_t *table_out, *len_out, *refs_out, *count;
  int32_t *src, *dst;        // pages to copy: [P / 2] (compact) or [n] (fork)
  uint64_t *masks;           // compact: [P / 64], and the sums after them; NULL: in LDS
};

// Sum over the workgroup of v in all threads before this one; total in `all`.
__device__ __forceinline__ int book_scan(int v, int &all) {
  __shared__ int part[kBookWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
  s += __builtin_amdgcn_update_dpp(0, s, 0x111, 0xf, 0xf, false); // row_shr 1, 2, 4, 8
  s += __builtin_amdgcn_update_dpp(0, s, 0x112, 0xf, 0xf, false);
  s += __builtin_amdgcn_update_dpp(0, s, 0x114, 0xf, 0xf, false);
  s += __builtin_amdgcn_update_dpp(0, s, 0x118, 0xf, 0xf, false);
  s += __builtin_amdgcn_update_dpp(0, s, 0x142, 0xa, 0xf, false); // row_bcast 15, 31
  s += __builtin_amdgcn_update_dpp(0, s, 0x143, 0xc, 0xf, false);
  __syncthreads(); // the last call's reads of `part`
  if (lane == 63)
    part[wave] = s;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kBookWaves; ++w) {
    if (w < wave)
      before += part[w];
    all += part[w];
  }
  return before + s - v;
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int shift) {
  return (tokens + (1ll << shift) - 1) >> shift;
}

// The free pages in ascending order, until `wanted` of them are found: f(rank, page) for each of
// those.  Returns how many there are (at most `wanted`); cut: the last of them (-1: none).
template <class F>
__device__ __forceinline__ int64_t book_free_pages(const int32_t *refs, int64_t P, int64_t wanted,
                                                   int64_t &cut, F f) {
  constexpr int N = 4, STEP = N * kBookThreads;
  __shared__ int last;
  if (threadIdx.x == 0)
    last = -1;
  int64_t found = 0;
  auto load = [&](int64_t base, int (&r)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t i = base + N * (int64_t)threadIdx.x + k;
      r[k] = refs[i < P ? i : 0];
      if (i >= P)
        r[k] = 1;
    }
  };
  int r[N], ahead[N];
  if (wanted > 0 && P > 0)
    load(0, r);
  for (int64_t base = 0; base < P && found < wanted; base += STEP) {
    if (base + STEP < P)
      load(base + STEP, ahead);
    int mine = 0, all;
#pragma unroll
    for (int k = 0; k < N; ++k)
      mine += r[k] == 0;
    int64_t rank = found + book_scan(mine, all);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (r[k] == 0) {
        const int page = (int)(base + N * (int64_t)threadIdx.x + k);
        if (rank < wanted)
          f(rank, page);
        if (rank == wanted - 1)
          last = page;
        ++rank;
      }
    found += all;
#pragma unroll
    for (int k = 0; k < N; ++k)
      r[k] = ahead[k];
  }
  __syncthreads();
  cut = found < wanted ? P - 1 : last;
  __syncthreads(); // `last` again
  return found < wanted ? found : wanted;
}

// New pages for the sequences.  Every workgroup sums the needs of all sequences, goes through the
// counts as far as there are pages wanted (a page that it finds goes straight to its place in
// the workgroup's rows, of which there may be none), and then writes its rows and its share of the
// counts: a free page up to the last one taken has been taken.
__global__ void __launch_bounds__(kBookThreads) page_reserve_kernel(BookArgs p) {
  __shared__ int pre[kBookRows + 1];   // pages that the sequences up to this row of ours want
  __shared__ int held_of[kBookRows];
  const int tid = threadIdx.x;
  const int64_t most = p.W << p.page_shift;
  auto after = [&](int64_t len, int64_t to) { // the length that a sequence gets
    const int64_t want = to < most ? to : most;
    return want > len ? want : len;
  };
  auto held = [&](int64_t len) {
    const int64_t h = pages_of(len > 0 ? len : 0, p.page_shift);
    return (int)(h < p.W ? h : p.W);
  };
  auto need = [&](int64_t len, int64_t to) {
    const int64_t h = pages_of(after(len, to), p.page_shift);
    const int x = (int)(h < p.W ? h : p.W) - held(len);
    return x > 0 ? x : 0;
  };
  int64_t nfree = 0, cut = -1, wanted = 0;
  // (once also where there are no rows for it: its share of the counts asks for the last page taken)
  int64_t s0 = (int64_t)blockIdx.x * p.rows;
  do {
    const int64_t left = p.S - s0;
    const int rows = (int)(left < 0 ? 0 : left < p.rows ? left : p.rows);
    int before = 0, all = 0, x;
    for (int64_t s = tid; s < p.S; s += kBookThreads) {
      const int v = need(p.len[s], p.new_len[s]);
      all += v;
      before += s < s0 ? v : 0;
    }
    book_scan(all, x);
    wanted = x;
    book_scan(before, x);
    const int64_t first_rank = x;
    int mine = 0;
    if (tid < rows) {
      const int64_t len = p.len[s0 + tid];
      mine = need(len, p.new_len[s0 + tid]);
      held_of[tid] = held(len);
    }
    const int at = book_scan(mine, x);
    if (tid < rows)
      pre[tid] = at;
    if (tid == 0)
      pre[rows] = x;
    const int ours = x;
    __syncthreads();
    nfree = book_free_pages(p.refs, p.P, wanted, cut, [&](int64_t rank, int page) {
      const int64_t r = rank - first_rank;
      if (r < 0 || r >= ours)
        return;
      int lo = 0, hi = rows; // pre[lo] <= r < pre[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (pre[mid] <= r)
          lo = mid;
        else
          hi = mid;
      }
      p.table_out[(s0 + lo) * p.W + held_of[lo] + (r - pre[lo])] = page;
    });
    // the other entries
    int tw = 64; // threads of a row
    while (tw < p.W && tw < kBookThreads)
      tw *= 2;
    for (int r = tid / tw; r < rows; r += kBookThreads / tw) {
      const int64_t row = (s0 + r) * p.W;
      const int h = held_of[r], fresh = pre[r + 1] - pre[r];
      const int64_t got = nfree - first_rank - pre[r]; // of `fresh`
      if (p.table_in_place) {
        for (int64_t w = (got > 0 ? got : 0) + (tid & (tw - 1)); w < fresh; w += tw)
          p.table_out[row + h + w] = -1;
        continue;
      }
      for (int64_t w = tid & (tw - 1); w < p.W; w += tw) {
        const int64_t k = w - h;
        if (k < 0 || k >= fresh)
          p.table_out[row + w] = p.table[row + w];
        else if (k >= got)
          p.table_out[row + w] = -1;
      }
    }
    __syncthreads(); // pre, held_of
    s0 += (int64_t)gridDim.x * p.rows;
  } while (s0 < p.S);
  if (p.refs_in_place) {
    for (int64_t i = tid; i <= cut; i += kBookThreads)
      if (p.refs[i] == 0)
        p.refs_out[i] = 1;
  } else {
    for (int64_t i = (int64_t)blockIdx.x * kBookThreads + tid; i < p.P;
         i += (int64_t)gridDim.x * kBookThreads) {
      const int r = p.refs[i];
      p.refs_out[i] = r == 0 && i <= cut ? 1 : r;
    }
  }
  // (len_out may be len, with one workgroup: every need has been summed)
  for (int64_t s = (int64_t)blockIdx.x * kBookThreads + tid; s < p.S;
       s += (int64_t)gridDim.x * kBookThreads)
    p.len_out[s] = (int32_t)after(p.len[s], p.new_len[s]);
  if (blockIdx.x == 0 && tid == 0)
    *p.count = (int32_t)(wanted - nfree);
}

// Workgroup 0 makes the children; the others copy the rows of who is not one.
__global__ void __launch_bounds__(kBookThreads) page_fork_kernel(BookArgs p) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    __shared__ int is_child[kBookRows];
    for (int64_t s0 = (int64_t)(blockIdx.x - 1) * p.rows; s0 < p.S;
         s0 += (int64_t)(gridDim.x - 1) * p.rows) {
      const int rows = (int)(p.S - s0 < p.rows ? p.S - s0 : p.rows);
      __syncthreads();
      for (int r = tid; r < rows; r += kBookThreads)
        is_child[r] = 0;
      __syncthreads();
      for (int i = tid; i < p.n; i += kBookThreads) {
        const int64_t a = p.parent[i], c = p.child[i];
        if (a >= 0 && a < p.S && c >= s0 && c < s0 + rows)
          is_child[c - s0] = 1;
      }
      __syncthreads();
      int tw = 64;
      while (tw < p.W && tw < kBookThreads)
        tw *= 2;
      for (int r = tid / tw; r < rows; r += kBookThreads / tw)
        if (!is_child[r])
          for (int64_t w = tid & (tw - 1); w < p.W; w += tw)
            p.table_out[(s0 + r) * p.W + w] = p.table[(s0 + r) * p.W + w];
      for (int r = tid; r < rows; r += kBookThreads)
        if (!is_child[r])
          p.len_out[s0 + r] = p.len[s0 + r];
    }
    return;
  }
  if (!p.refs_in_place)
    for (int64_t i = tid; i < p.P; i += kBookThreads)
      p.refs_out[i] = p.refs[i];
  // src[i], dst[i]: the last page of child i's parent and its copy (-1: none).  A batch of children
  // is looked up once, into LDS.
  struct Child {
    int a, c, len, rank; // parent (-1: the pair is skipped), child, rank of the page it wants or -1
  };
  __shared__ Child kids[kBookThreads];
  auto look_up = [&](int base, int &last, int64_t before) {
    const int i = base + tid;
    Child k{-1, 0, 0, -1};
    int open = 0, all;
    last = -1;
    if (i < p.n) {
      const int a = p.parent[i], c = p.child[i];
      if (a >= 0 && a < p.S && c >= 0 && c < p.S) {
        const int len = p.len[a];
        k.a = a, k.c = c, k.len = len > 0 ? len : 0;
        const int64_t used = pages_of(k.len, p.page_shift);
        open = (k.len & ((1 << p.page_shift) - 1)) != 0 && used <= p.W;
        if (open)
          last = p.table[a * p.W + used - 1];
      }
    }
    const int at = book_scan(open, all);
    k.rank = open ? (int)before + at : -1;
    kids[tid] = k;
    return all;
  };
  int64_t wanted = 0;
  for (int base = 0; base < p.n; base += kBookThreads) {
    int last;
    wanted += look_up(base, last, wanted);
    if (base + tid < p.n)
      p.src[base + tid] = last;
  }
  int64_t cut;
  const int64_t nfree = book_free_pages(p.refs, p.P, wanted, cut, [&](int64_t rank, int page) {
    p.src[p.n + rank] = page; // (src has place for 2 n)
    p.refs_out[page] = 1;
  });
  int tw = 64;
  while (tw < p.W && tw < kBookThreads)
    tw *= 2;
  const int per = kBookThreads / tw;
  int64_t before = 0;
  for (int base = 0; base < p.n; base += kBookThreads) {
    if (p.n > kBookThreads) { // (else kids holds them)
      int last;
      __syncthreads();
      before += look_up(base, last, before);
    }
    __syncthreads();
    if (base + tid < p.n) {
      const int rank = kids[tid].rank;
      kids[tid].rank = rank < 0 ? -2 : rank < nfree ? p.src[p.n + rank] : -1; // the page; -2: none
      p.dst[base + tid] = kids[tid].rank < 0 ? -1 : kids[tid].rank;
    }
    __syncthreads();
    const int m = p.n - base < kBookThreads ? p.n - base : kBookThreads;
    constexpr int N = 4; // rows under way
    for (int i0 = tid / tw; i0 < m; i0 += N * per)
      for (int64_t w = tid & (tw - 1); w < p.W; w += tw) {
        int page[N];
        bool shared[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int i = i0 + k * per;
          const Child kid = kids[i < m ? i : 0];
          const int64_t used = pages_of(kid.len, p.page_shift);
          shared[k] = i < m && kid.a >= 0 && w < used;
          page[k] = -1;
          if (shared[k]) {
            if (kid.rank != -2 && w == used - 1)
              page[k] = kid.rank, shared[k] = false;
            else
              page[k] = p.table[kid.a * p.W + w];
          }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int i = i0 + k * per;
          if (i >= m || kids[i].a < 0)
            continue;
          if (shared[k] && page[k] >= 0 && page[k] < p.P)
            atomicAdd(&p.refs_out[page[k]], 1);
          p.table_out[kids[i].c * p.W + w] = page[k];
        }
      }
    if (base + tid < p.n && kids[tid].a >= 0)
      p.len_out[kids[tid].c] = kids[tid].len;
  }
  if (tid == 0)
    *p.count = (int32_t)(wanted - nfree);
}

__global__ void __launch_bounds__(256) book_copy_kernel(int32_t *to, const int32_t *from, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    to[i] = from[i];
}

// refs_out holds the counts already.  A row's entries, then its length (which may be in place).
__global__ void __launch_bounds__(kBookThreads) page_free_kernel(BookArgs p) {
  const int tid = threadIdx.x;
  int tw = 64;
  while (tw < p.W && tw < kBookThreads)
    tw *= 2;
  const int per = kBookThreads / tw;
  for (int64_t s0 = (int64_t)blockIdx.x * per; s0 < p.S; s0 += (int64_t)gridDim.x * per) {
    const int64_t s = s0 + tid / tw;
    const bool on = s < p.S;
    const int len = on ? p.len[s] : 0;
    const bool drop = on && p.drop[s];
    const int64_t used = pages_of(len > 0 ? len : 0, p.page_shift);
    for (int64_t w = tid & (tw - 1); on && w < p.W; w += tw) {
      if (drop) {
        const int32_t page = p.table[s * p.W + w];
        if (w < used && page >= 0 && page < p.P)
          atomicSub(&p.refs_out[page], 1);
        p.table_out[s * p.W + w] = -1;
      } else if (!p.table_in_place) {
        p.table_out[s * p.W + w] = p.table[s * p.W + w];
      }
    }
    __syncthreads(); // len_out may be len
    if (on && (tid & (tw - 1)) == 0)
      p.len_out[s] = drop ? 0 : len;
  }
}

// The same in one launch, where the table is small and nothing that all read is written: every
// workgroup goes through the whole table and counts, in LDS, what is given back of its own
// kFreePages pages.  Bound by its two trips to memory: 8 rows of 16 take 2.1 us (the copy and the
// atomics 3.8), 64 of 64, the largest, 3.8 (4.3); in a stream of calls 6.9 (9.7), the host's launches.
// With 32 entries a thread it took 7.7 (4.8).
constexpr int kFreePages = kBookThreads, kFreeEach = 8, kFreeEntries = kFreeEach * kBookThreads;

__global__ void __launch_bounds__(kBookThreads) page_free_small_kernel(BookArgs p) {
  __shared__ int used[kFreeEntries]; // pages of a row that is dropped; -1: it is not
  __shared__ int gone[kFreePages];
  const int tid = threadIdx.x, first = (int)blockIdx.x * kFreePages;
  const int W = (int)p.W, entries = p.S * W;
  int page[kFreeEach];
#pragma unroll
  for (int k = 0; k < kFreeEach; ++k) {
    const int i = tid + k * kBookThreads;
    page[k] = p.table[i < entries ? i : 0];
  }
  const int refs = p.refs[first + tid < p.P ? first + tid : 0];
  gone[tid] = 0;
  for (int s = tid; s < p.S; s += kBookThreads) {
    const int len = p.len[s];
    const bool drop = p.drop[s];
    const int64_t n = pages_of(len > 0 ? len : 0, p.page_shift);
    used[s] = !drop ? -1 : n < W ? (int)n : W;
    if (blockIdx.x == 0)
      p.len_out[s] = drop ? 0 : len;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kFreeEach; ++k) {
    const int i = tid + k * kBookThreads;
    if (i < entries) {
      const int row = i / W, n = used[row];
      if (i - row * W < n && page[k] >= first && page[k] - first < kFreePages)
        atomicAdd(&gone[page[k] - first], 1);
      if (k % gridDim.x == blockIdx.x)
        p.table_out[i] = n >= 0 ? -1 : page[k];
    }
  }
  __syncthreads();
  if (first + tid < p.P)
    p.refs_out[first + tid] = refs - gone[tid];
}

// With U pages in use: which pages are, as bits, and how many of them lie before each 64, from which
// every workgroup finds by itself where a page goes and where it came from.
constexpr int kBookMasks = 4096; // 64 pages each, in LDS

__global__ void __launch_bounds__(kBookThreads) page_compact_kernel(BookArgs p) {
  __shared__ uint64_t lds_masks[kBookMasks];
  __shared__ int lds_sums[kBookMasks + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int groups = (int)(((int64_t)p.P + 63) / 64);
  uint64_t *const masks = p.masks ? p.masks : lds_masks;
  int *const sums = p.masks ? reinterpret_cast<int *>(p.masks + groups) : lds_sums;
  constexpr int N = 8; // groups a wave has under way
  for (int g0 = wave * N; g0 < groups; g0 += kBookWaves * N) {
    int r[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t i = 64 * (int64_t)(g0 + k) + lane;
      r[k] = p.refs[i < p.P ? i : 0];
      if (i >= p.P)
        r[k] = 0;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint64_t live = __ballot(r[k] > 0);
      if (lane == 0 && g0 + k < groups)
        masks[g0 + k] = live;
    }
  }
  __syncthreads();
  int used = 0;
  for (int base = 0; base < groups; base += kBookThreads) {
    const int g = base + tid;
    int all;
    const int at = book_scan(g < groups ? __popcll(masks[g]) : 0, all);
    if (g < groups)
      sums[g] = used + at;
    used += all;
  }
  if (tid == 0)
    sums[groups] = used;
  __syncthreads();
  auto live_below = [&](int page) {
    const int g = page >> 6, b = page & 63;
    return g >= groups ? used : sums[g] + __popcll(masks[g] & ((1ull << b) - 1));
  };
  // the k-th page that is in use (or, `free`, that is not)
  auto select = [&](int k, bool free) {
    int lo = 0, hi = groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      const int at = free ? (int)(64 * (int64_t)mid - sums[mid]) : sums[mid];
      if (at <= k)
        lo = mid;
      else
        hi = mid;
    }
    k -= free ? (int)(64 * (int64_t)lo - sums[lo]) : sums[lo];
    const uint64_t m = free ? ~masks[lo] : masks[lo];
    int at = 0; // the k-th bit of m
#pragma unroll
    for (int d = 32; d; d /= 2) {
      const int c = __popcll((m >> at) & ((1ull << d) - 1));
      if (c <= k)
        k -= c, at += d;
    }
    return 64 * lo + at;
  };
  const int stay = live_below(used), movers = used - stay; // pages in use below U, and past it
  const int64_t first = (int64_t)blockIdx.x * kBookThreads + tid,
                step = (int64_t)gridDim.x * kBookThreads;
  for (int64_t m = first; m < movers; m += step) {
    const int a = select(stay + (int)m, false), b = select((int)m, true);
    p.src[m] = a, p.dst[m] = b;
    if (p.refs_in_place) {
      p.refs_out[b] = p.refs[a];
      p.refs_out[a] = 0;
    }
  }
  if (!p.refs_in_place)
    for (int64_t i = first; i < p.P; i += step) {
      const bool live = masks[i >> 6] >> (i & 63) & 1;
      int from = (int)i;
      if (i < used && !live)
        from = select(stay + (int)i - live_below((int)i), false);
      const int r = p.refs[from];
      p.refs_out[i] = i >= used && live ? 0 : r;
    }
  const int64_t entries = p.S * p.W;
  for (int64_t i = first; i < entries; i += step) {
    int page = p.table[i];
    // (an entry may name a page that is not in use: it stays)
    if (page >= used && page < p.P && (masks[page >> 6] >> (page & 63) & 1))
      page = select(live_below(page) - stay, true);
    p.table_out[i] = page;
  }
  if (blockIdx.x == 0 && tid == 0)
    *p.count = movers;
}

struct PageCopyArgs {
  const int32_t *src, *dst;
  const int32_t *count; // pages to copy; NULL: n
  int64_t n, P;
  int32_t caches;
  uint8_t *base[TX_PAGE_CACHES];
  int64_t stride[TX_PAGE_CACHES], bytes[TX_PAGE_CACHES];
};

// blockIdx.y: the cache.  Pieces of 16 KiB (256 threads x 4 x 16 bytes, all four loads before
// the stores), non-temporal: 32 KiB pages of 4 caches at 5.7 TB/s read and written (60 us for 246 MB with
// the books; 68 through the caches).  Bound by memory.
__global__ void __launch_bounds__(256) page_copy_kernel(PageCopyArgs p) {
  const int c = blockIdx.y;
  const int64_t bytes = p.bytes[c], stride = p.stride[c];
  uint8_t *const base = p.base[c];
  const uint32_t n = (uint32_t)(p.count ? *p.count : p.n);
  const uint32_t pieces = (uint32_t)((bytes + 16383) / 16384);
  if (pieces == 0)
    return;
  uint32_t i = blockIdx.x / pieces, at_piece = blockIdx.x - i * pieces;
  const uint32_t step_i = gridDim.x / pieces, step_p = gridDim.x - step_i * pieces;
  while (i < n) {
    const int64_t a = p.src[i], b = p.dst[i];
    if (a >= 0 && a < p.P && b >= 0 && b < p.P && a != b) {
      const int64_t at = (int64_t)at_piece * 16384 + threadIdx.x * 16;
      u32x4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at + 4096 * k < bytes)
          x[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(base + a * stride + at + 4096 * k));
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (at + 4096 * k < bytes)
          __builtin_nontemporal_store(x[k], reinterpret_cast<u32x4 *>(base + b * stride + at + 4096 * k));
    }
    i += step_i, at_piece += step_p;
    if (at_piece >= pieces)
      at_piece -= pieces, ++i;
  }
}

} // namespace txk
