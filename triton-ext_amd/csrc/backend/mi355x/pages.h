// The books of a paged cache (page table, lengths, reference counts) and the moves
// of its pages.
//
// The books are integers of a few hundred KiB at most: one workgroup of 1024
// threads goes through them with prefix sums, so that free pages are taken in
// ascending order whatever the timing.  Pages are copied by a kernel of their own
// that takes its list (and, compacting, its length) from device memory.
#pragma once

#include <hip/hip_runtime.h>

#include "tile_common.h"
#include "triton_ext/tx_cache.h"

namespace txk {

constexpr int kBookThreads = 1024;

struct BookArgs {
  int64_t S, W, P, n;
  int32_t page_shift;
  const int32_t *table, *len, *refs;
  const int32_t *new_len, *parent, *child;
  const uint8_t *drop;
  int32_t *table_out, *len_out, *refs_out, *count;
  int32_t *free_list; // [P]: free pages in ascending order; compact: the map of pages
  int32_t *src, *dst; // [P] (compact) or [n] (fork): pages to copy
  int32_t *prefix;    // [S + 1] (reserve)
};

// Sum over the workgroup of v in all threads before this one; total in `all`.
__device__ __forceinline__ int book_scan(int v, int &all) {
  __shared__ int part[kBookThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(s, d);
    if (lane >= d)
      s += o;
  }
  __syncthreads(); // the last call's reads of `part`
  if (lane == 63)
    part[wave] = s;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kBookThreads / 64; ++w) {
    if (w < wave)
      before += part[w];
    all += part[w];
  }
  return before + s - v;
}

// The free pages in ascending order into free_list; returns how many there are.
__device__ __forceinline__ int64_t book_free_list(const BookArgs &p) {
  int64_t free_pages = 0;
  for (int64_t base = 0; base < p.P; base += kBookThreads) {
    const int64_t i = base + threadIdx.x;
    const int is_free = i < p.P && p.refs[i] == 0;
    int all;
    const int at = book_scan(is_free, all);
    if (is_free)
      p.free_list[free_pages + at] = (int32_t)i;
    free_pages += all;
  }
  return free_pages;
}

__device__ __forceinline__ void book_copy(int32_t *to, const int32_t *from, int64_t n) {
  if (to != from)
    for (int64_t i = threadIdx.x; i < n; i += kBookThreads)
      to[i] = from[i];
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int shift) {
  return (tokens + (1ll << shift) - 1) >> shift;
}

__global__ void __launch_bounds__(kBookThreads) page_reserve_kernel(BookArgs p) {
  const int64_t nfree = book_free_list(p);
  const int64_t most = p.W << p.page_shift;
  auto after = [&](int64_t s) { // the length that sequence s gets
    const int64_t want = p.new_len[s] < most ? p.new_len[s] : most;
    return want > p.len[s] ? want : (int64_t)p.len[s];
  };
  auto held = [&](int64_t s) {
    const int64_t h = pages_of(p.len[s] > 0 ? p.len[s] : 0, p.page_shift);
    return h < p.W ? h : p.W;
  };
  int64_t wanted = 0;
  for (int64_t base = 0; base < p.S; base += kBookThreads) {
    const int64_t s = base + threadIdx.x;
    int need = 0;
    if (s < p.S) {
      const int64_t to = pages_of(after(s), p.page_shift);
      need = (int)((to < p.W ? to : p.W) - held(s));
      need = need > 0 ? need : 0;
    }
    int all;
    const int at = book_scan(need, all);
    if (s < p.S)
      p.prefix[s] = (int32_t)(wanted + at);
    wanted += all;
  }
  if (threadIdx.x == 0)
    p.prefix[p.S] = (int32_t)wanted;
  book_copy(p.refs_out, p.refs, p.P);
  __syncthreads();
  for (int64_t i = threadIdx.x; i < p.S * p.W; i += kBookThreads) {
    const int64_t s = i / p.W, w = i % p.W, first = held(s);
    const int64_t rank = p.prefix[s] + w - first;
    if (w < first || rank >= p.prefix[s + 1]) {
      p.table_out[i] = p.table[i];
      continue;
    }
    const int32_t page = rank < nfree ? p.free_list[rank] : -1;
    p.table_out[i] = page;
    if (page >= 0)
      p.refs_out[page] = 1;
  }
  if (threadIdx.x == 0)
    *p.count = (int32_t)(wanted > nfree ? wanted - nfree : 0);
  __syncthreads(); // len_out may be len
  for (int64_t base = 0; base < p.S; base += kBookThreads) {
    const int64_t s = base + threadIdx.x;
    if (s < p.S)
      p.len_out[s] = (int32_t)after(s);
  }
}

__global__ void __launch_bounds__(kBookThreads) page_fork_kernel(BookArgs p) {
  const int64_t nfree = book_free_list(p);
  book_copy(p.refs_out, p.refs, p.P);
  book_copy(p.table_out, p.table, p.S * p.W);
  book_copy(p.len_out, p.len, p.S);
  __syncthreads();
  int64_t wanted = 0;
  // src[i], dst[i]: the last page of child i's parent and its copy (-1: none)
  for (int64_t base = 0; base < p.n; base += kBookThreads) {
    const int64_t i = base + threadIdx.x;
    int open = 0, last = -1;
    if (i < p.n) {
      const int64_t a = p.parent[i], c = p.child[i];
      if (a >= 0 && a < p.S && c >= 0 && c < p.S) {
        const int64_t len = p.len[a] > 0 ? p.len[a] : 0, used = pages_of(len, p.page_shift);
        open = (len & ((1 << p.page_shift) - 1)) != 0 && used <= p.W;
        if (open)
          last = p.table[a * p.W + used - 1];
      }
    }
    int all;
    const int at = book_scan(open, all);
    if (i < p.n) {
      const int32_t page = open && wanted + at < nfree ? p.free_list[wanted + at] : -1;
      p.src[i] = last;
      p.dst[i] = page;
      if (page >= 0)
        p.refs_out[page] = 1;
    }
    wanted += all;
  }
  __syncthreads();
  for (int64_t j = threadIdx.x; j < p.n * p.W; j += kBookThreads) {
    const int64_t i = j / p.W, w = j % p.W;
    const int64_t a = p.parent[i], c = p.child[i];
    if (a < 0 || a >= p.S || c < 0 || c >= p.S)
      continue;
    const int64_t len = p.len[a] > 0 ? p.len[a] : 0, used = pages_of(len, p.page_shift);
    const bool open = (len & ((1 << p.page_shift) - 1)) != 0;
    int32_t page = -1;
    if (w < used) {
      page = p.table[a * p.W + w];
      if (open && w == used - 1)
        page = p.dst[i];
      else if (page >= 0 && page < p.P)
        atomicAdd(&p.refs_out[page], 1);
    }
    p.table_out[c * p.W + w] = page;
    if (w == 0)
      p.len_out[c] = (int32_t)len;
  }
  if (threadIdx.x == 0)
    *p.count = (int32_t)(wanted > nfree ? wanted - nfree : 0);
}

__global__ void __launch_bounds__(kBookThreads) page_free_kernel(BookArgs p) {
  book_copy(p.refs_out, p.refs, p.P);
  __syncthreads();
  for (int64_t i = threadIdx.x; i < p.S * p.W; i += kBookThreads) {
    const int64_t s = i / p.W, w = i % p.W;
    const int32_t page = p.table[i];
    if (p.drop[s]) {
      if (w < pages_of(p.len[s] > 0 ? p.len[s] : 0, p.page_shift) && page >= 0 && page < p.P)
        atomicSub(&p.refs_out[page], 1);
      p.table_out[i] = -1;
    } else {
      p.table_out[i] = page;
    }
  }
  __syncthreads(); // len_out may be len
  for (int64_t s = threadIdx.x; s < p.S; s += kBookThreads)
    p.len_out[s] = p.drop[s] ? 0 : p.len[s];
}

__global__ void __launch_bounds__(kBookThreads) page_compact_kernel(BookArgs p) {
  int used = 0, n;
  for (int64_t base = 0; base < p.P; base += kBookThreads) {
    const int64_t i = base + threadIdx.x;
    book_scan(i < p.P && p.refs[i] > 0, n);
    used += n;
  }
  // holes below `used` and used pages from there on, as many of the one as of the other
  int64_t holes = 0, movers = 0;
  for (int64_t base = 0; base < p.P; base += kBookThreads) {
    const int64_t i = base + threadIdx.x;
    const bool live = i < p.P && p.refs[i] > 0;
    const int hole = i < used && !live, mover = i >= used && live;
    int all;
    const int at = book_scan(hole, all);
    if (hole)
      p.dst[holes + at] = (int32_t)i;
    holes += all;
    const int at2 = book_scan(mover, all);
    if (mover)
      p.src[movers + at2] = (int32_t)i;
    movers += all;
    if (i < p.P)
      p.free_list[i] = (int32_t)i;
  }
  book_copy(p.refs_out, p.refs, p.P);
  __syncthreads();
  for (int64_t i = threadIdx.x; i < movers; i += kBookThreads) {
    const int32_t a = p.src[i], b = p.dst[i];
    p.free_list[a] = b;
    p.refs_out[b] = p.refs_out[a];
    p.refs_out[a] = 0;
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < p.S * p.W; i += kBookThreads) {
    const int32_t page = p.table[i];
    p.table_out[i] = page >= 0 && page < p.P ? p.free_list[page] : page;
  }
  if (threadIdx.x == 0)
    *p.count = (int32_t)movers;
}

struct PageCopyArgs {
  const int32_t *src, *dst;
  const int32_t *count; // pages to copy; NULL: n
  int64_t n, P;
  int32_t caches;
  uint8_t *base[TX_PAGE_CACHES];
  int64_t stride[TX_PAGE_CACHES], bytes[TX_PAGE_CACHES];
};

// blockIdx.y: the cache.  Pieces of 4 KiB (256 threads x 16 bytes).
__global__ void __launch_bounds__(256) page_copy_kernel(PageCopyArgs p) {
  const int c = blockIdx.y;
  const int64_t n = p.count ? *p.count : p.n;
  const int64_t pieces = (p.bytes[c] + 4095) / 4096;
  for (int64_t w = blockIdx.x; w < n * pieces; w += gridDim.x) {
    const int64_t i = w / pieces, at = (w % pieces) * 4096 + threadIdx.x * 16;
    const int64_t a = p.src[i], b = p.dst[i];
    if (a < 0 || a >= p.P || b < 0 || b >= p.P || a == b || at >= p.bytes[c])
      continue;
    *reinterpret_cast<u32x4 *>(p.base[c] + b * p.stride[c] + at) =
        *reinterpret_cast<const u32x4 *>(p.base[c] + a * p.stride[c] + at);
  }
}

} // namespace txk
