// What the launch layers of the paged cache share (MI355xCache.hip, MI355xCache4.hip): arithmetic of
// grids, and the checks of descriptors.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>

#include "launch_common.h"
#include "rotary.h"
#include "triton_ext/tx_cache.h"

namespace {

using namespace txk;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool pow2(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }
int log2of(int64_t x) {
  int s = 0;
  while ((1ll << s) < x)
    ++s;
  return s;
}
int64_t sizeOf(int32_t t) { return t == TX_F32 ? 4 : t == TX_F8E4M3 ? 1 : 2; }
bool aligned(const void *p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// One tensor of tokens: strides of the dimensions that have more than one element
// must not be negative, and, where it is written, not 0.
int checkStrides(const char *name, int64_t rows, int64_t sr, int64_t heads, int64_t sh,
                 int64_t head_dim, bool written) {
  if (sr < 0 || sh < 0)
    return fail(TX_ERR_INVALID, "%s: negative stride", name);
  if (written && ((rows > 1 && sr < head_dim) || (heads > 1 && sh < head_dim)))
    return fail(TX_ERR_INVALID, "%s: rows that overlap (strides %lld, %lld for %lld elements)",
                name, (long long)sr, (long long)sh, (long long)head_dim);
  return TX_OK;
}

// The largest power of two up to `most` that divides every one of n.
int commonVec(int most, std::initializer_list<int64_t> n) {
  int v = most;
  for (int64_t x : n)
    while (x % v)
      v /= 2;
  return v;
}

// Threads that share a token's heads: enough to give every CU 32 waves (256 x 32 x 64
// threads), fewer where the tokens alone do, since a thread's sines cost about what two heads do.
int headLanes(int64_t tokens, int64_t items, int64_t heads) {
  const int64_t want = 256 * 32 * 64;
  int64_t lanes = cdiv(want, std::max<int64_t>(tokens * items, 1));
  // (a batch of heads each)
  lanes = std::max<int64_t>(std::min(lanes, cdiv(heads, tokens * items * heads > want ? kHeadBatch : 1)), 1);
  return (int)std::min<int64_t>(lanes, std::max<int64_t>(heads, 1));
}
// Workgroups of 256 for tokens of so many threads (RotaryPlace).
int64_t tokenGrid(int64_t tokens, int64_t token_threads) {
  return token_threads <= 256 ? cdiv(tokens, 256 / token_threads) : tokens * cdiv(token_threads, 256);
}

// What paged_append and paged_attention ask alike of the cache and its tables.
// packed: a cache of TX_F4E2M1 (its own entry points).
template <class D> int checkPaged(const D &d, int flag, bool packed = false) {
  if (d.T < 0 || d.B < 0 || d.pages < 0 || d.table_width < 0 || d.Hq < 0 || d.Hkv < 0)
    return fail(TX_ERR_INVALID, "negative extent");
  if (d.T > INT32_MAX || d.B > INT32_MAX / 2 || d.pages > INT32_MAX || d.table_width > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "extents above 2^31");
  if (d.dtype != TX_F16 && d.dtype != TX_BF16)
    return fail(TX_ERR_UNSUPPORTED, "dtype %d: fp16 and bf16 are implemented", d.dtype);
  if (packed ? d.cache_type != TX_F4E2M1
             : d.cache_type != d.dtype && d.cache_type != TX_F8E4M3)
    return fail(TX_ERR_UNSUPPORTED, packed ? "cache type %d: e2m1" : "cache type %d: that of the tokens, or fp8 e4m3",
                d.cache_type);
  if (!pow2(d.page_size) || d.page_size > 65536)
    return fail(TX_ERR_UNSUPPORTED, "page_size %d: a power of two up to 65536", d.page_size);
  if (d.head_dim < 1)
    return fail(TX_ERR_INVALID, "head_dim %d", d.head_dim);
  if ((flag | d.ragged) & ~1)
    return fail(TX_ERR_INVALID, "flags must be 0 or 1");
  if (!d.ragged && d.T != d.B)
    return fail(TX_ERR_INVALID, "%lld tokens of %lld sequences: cu_q is needed", (long long)d.T,
                (long long)d.B);
  if (d.T > 0 && d.B == 0)
    return fail(TX_ERR_INVALID, "new tokens, but no sequence");
  if (d.table_s < 0 || (d.B > 1 && d.table_s < d.table_width))
    return fail(TX_ERR_INVALID, "page_table rows overlap");
  return TX_OK;
}
int checkCache(const char *name, int64_t pages, int64_t sp, int64_t page_size, int64_t st,
               int64_t heads, int64_t sh, int64_t head_dim) {
  if (sp < 0 || st < 0 || sh < 0)
    return fail(TX_ERR_INVALID, "%s: negative stride", name);
  if ((pages > 1 && sp < head_dim) || (page_size > 1 && st < head_dim) ||
      (heads > 1 && sh < head_dim))
    return fail(TX_ERR_INVALID, "%s: rows that overlap", name);
  return TX_OK;
}

constexpr int64_t kAttnCounters = 65536; // the arrival counters that every workspace begins with

// The dims that a head is computed in.
int attnDims(int head_dim) {
  return head_dim <= 64 ? 64 : head_dim <= 96 ? 96 : head_dim <= 128 ? 128 : 256;
}

} // namespace
