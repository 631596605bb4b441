// Launch layer of the paged cache: rotary positions, new tokens into the cache,
// attention over it, and its pages (tx_cache.h).

#include <algorithm>
#include <cmath>
#include <cstring>

#include "launch_common.h"
#include "paged_attn.h"
#include "pages.h"
#include "rotary.h"
#include "triton_ext/tx_cache.h"

using namespace txk;

namespace txk {
typedef void (*PagedAttnFn)(PagedAttnArgs);
// [64, 96, 128, 256 dims][bf16][e4m3 cache] (kernels_paged_*.hip)
extern const PagedAttnFn kPagedAttnSplit16[4][2][2], kPagedAttnSplit[4][2][2], kPagedAttnRows[4][2][2];
} // namespace txk

namespace {

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

// Items of a head (rotary.h): runs of `vec` elements or pairs of them.
int itemsOf(int head_dim, int rot, int vec, bool interleaved) {
  const int pairs = rot == 0 ? 0 : interleaved ? rot / (vec > 1 ? vec : 2) : rot / 2 / vec;
  return pairs + (head_dim - rot) / vec;
}
int vecOf(int most, int head_dim, int rot, bool interleaved) {
  return interleaved ? commonVec(most, {head_dim, rot ? rot : most})
                     : commonVec(most, {head_dim, rot ? rot / 2 : most});
}

template <class T> void rotaryKernels(void (*(&k)[2][4])(RotaryArgs)) {
  k[0][0] = rotary_kernel<T, 1, false>, k[0][1] = rotary_kernel<T, 2, false>;
  k[0][2] = rotary_kernel<T, 4, false>;
  k[1][0] = rotary_kernel<T, 1, true>, k[1][1] = rotary_kernel<T, 2, true>;
  k[1][2] = rotary_kernel<T, 4, true>;
  if constexpr (sizeof(T) == 2) {
    k[0][3] = rotary_kernel<T, 8, false>;
    k[1][3] = rotary_kernel<T, 8, true>;
  }
}

} // namespace

// ---------------------------------------------------------------------------
// Rotary positions
// ---------------------------------------------------------------------------

extern "C" TX_API int tx_rotary_plan_create(const tx_rotary_desc *desc, tx_rotary_plan *plan) {
  clearError();
  if (!desc || !plan)
    return fail(TX_ERR_INVALID, "descriptor or plan is NULL");
  const tx_rotary_desc &d = *desc;
  if (d.Z < 0 || d.N < 0 || d.H < 0)
    return fail(TX_ERR_INVALID, "negative extent Z=%lld N=%lld H=%lld", (long long)d.Z,
                (long long)d.N, (long long)d.H);
  if (d.dtype != TX_F32 && d.dtype != TX_F16 && d.dtype != TX_BF16)
    return fail(TX_ERR_UNSUPPORTED, "dtype %d: fp32, fp16 and bf16 are implemented", d.dtype);
  if (d.head_dim < 1 || d.head_dim > 65536 || d.rot_dim < 2 || d.rot_dim > d.head_dim ||
      d.rot_dim % 2)
    return fail(TX_ERR_INVALID, "rot_dim %d of head_dim %d: an even number of its dims", d.rot_dim,
                d.head_dim);
  if ((d.interleaved | d.inverse) & ~1)
    return fail(TX_ERR_INVALID, "interleaved and inverse must be 0 or 1");
  if (d.pos_bits != 32 && d.pos_bits != 64)
    return fail(TX_ERR_INVALID, "pos_bits %d: positions are int32 or int64", d.pos_bits);
  if (!std::isfinite(d.scale) || d.reserved != 0 || d.pos_sz < 0)
    return fail(TX_ERR_INVALID, "scale must be finite, reserved 0 and pos_sz not negative");
  const int64_t lim = (int64_t)1 << 40;
  if (d.Z > lim || d.N > lim || d.H > INT32_MAX || (d.N > 0 && d.Z > lim / d.N))
    return fail(TX_ERR_UNSUPPORTED, "extents above 2^40");
  int rc = checkStrides("x", d.N, d.x_sn, d.H, d.x_sh, d.head_dim, false);
  if (rc == TX_OK) rc = checkStrides("out", d.N, d.o_sn, d.H, d.o_sh, d.head_dim, true);
  if (rc == TX_OK) rc = checkStrides("x", d.Z, d.x_sz, 1, 0, d.head_dim, false);
  if (rc == TX_OK) rc = checkStrides("out", d.Z, d.o_sz, 1, 0, d.head_dim, true);
  if (rc != TX_OK)
    return rc;
  std::memset(plan, 0, sizeof(*plan));
  plan->desc = d;
  const double n = (double)d.Z * d.N * d.H;
  plan->flops = 3.0 * n * d.rot_dim;
  plan->bytes = 2.0 * n * d.head_dim * sizeOf(d.dtype);
  const int most = (int)(16 / sizeOf(d.dtype));
  plan->vec = commonVec(vecOf(most, d.head_dim, d.rot_dim, d.interleaved),
                        {d.x_sz, d.x_sn, d.x_sh, d.o_sz, d.o_sn, d.o_sh});
  const int64_t items = itemsOf(d.head_dim, d.rot_dim, plan->vec, d.interleaved);
  plan->head_lanes = (int)std::min<int64_t>(headLanes(d.Z * d.N, items, d.H), 65535);
  plan->block_threads = 256;
  const bool token_fast = d.x_sh > d.x_sn && d.N > 1;
  const int64_t per = token_fast ? items : items * plan->head_lanes;
  // (a base that is less aligned than vec runs at vec 1, with 16 times the threads at most)
  if (tokenGrid(d.Z * d.N, per) * 32 > INT32_MAX || items * plan->head_lanes > INT32_MAX / 32)
    return fail(TX_ERR_UNSUPPORTED, "grid above 2^31");
  plan->grid_x = d.H == 0 ? 0 : (int32_t)tokenGrid(d.Z * d.N, per);
  return TX_OK;
}

extern "C" TX_API int tx_rotary_launch(const tx_rotary_plan *plan, const void *x,
                                       const void *positions, const float *inv_freq, void *out,
                                       void *stream) {
  clearError();
  if (!plan)
    return fail(TX_ERR_INVALID, "plan is NULL");
  tx_rotary_plan again;
  const int rc = tx_rotary_plan_create(&plan->desc, &again);
  if (rc != TX_OK)
    return rc;
  if (std::memcmp(&again, plan, sizeof again) != 0)
    return fail(TX_ERR_INVALID, "the plan does not follow from its descriptor");
  if (plan->grid_x == 0)
    return TX_OK;
  const tx_rotary_desc &d = plan->desc;
  if (!x || !positions || !inv_freq || !out)
    return fail(TX_ERR_INVALID, "NULL tensor pointer");
  const int64_t e = sizeOf(d.dtype);
  if (!aligned(x, e) || !aligned(out, e) || !aligned(positions, d.pos_bits / 8) ||
      !aligned(inv_freq, 4))
    return fail(TX_ERR_INVALID, "a tensor is not aligned to its elements");
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  int vec = plan->vec, lanes = plan->head_lanes;
  if (!aligned(x, vec * e) || !aligned(out, vec * e)) {
    vec = 1;
    lanes = (int)std::min<int64_t>(
        headLanes(d.Z * d.N, itemsOf(d.head_dim, d.rot_dim, 1, d.interleaved), d.H), 65535);
  }
  RotaryArgs a;
  a.x = x, a.pos = positions, a.inv_freq = inv_freq, a.out = out;
  a.N = d.N, a.tokens = d.Z * d.N, a.pos_sz = d.pos_sz;
  a.x_sz = d.x_sz, a.x_sn = d.x_sn, a.x_sh = d.x_sh;
  a.o_sz = d.o_sz, a.o_sn = d.o_sn, a.o_sh = d.o_sh;
  a.H = (int32_t)d.H, a.head_dim = d.head_dim, a.rot = d.rot_dim;
  a.items = itemsOf(d.head_dim, d.rot_dim, vec, d.interleaved);
  a.token_fast = d.x_sh > d.x_sn && d.N > 1;
  a.token_threads = a.token_fast ? a.items : a.items * lanes;
  a.head_lanes = lanes, a.pos64 = d.pos_bits == 64, a.inverse = d.inverse, a.scale = d.scale;
  void (*fn[2][4])(RotaryArgs) = {};
  if (d.dtype == TX_F32)
    rotaryKernels<float>(fn);
  else if (d.dtype == TX_F16)
    rotaryKernels<_Float16>(fn);
  else
    rotaryKernels<__bf16>(fn);
  const int64_t grid = tokenGrid(d.Z * d.N, a.token_threads);
  hipLaunchKernelGGL(fn[d.interleaved][log2of(vec)],
                     dim3((uint32_t)grid, a.token_fast ? (uint32_t)lanes : 1), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}

// ---------------------------------------------------------------------------
// New tokens into the cache
// ---------------------------------------------------------------------------

namespace {

// What paged_append and paged_attention ask alike of the cache and its tables.
template <class D> int checkPaged(const D &d, int flag) {
  if (d.T < 0 || d.B < 0 || d.pages < 0 || d.table_width < 0 || d.Hq < 0 || d.Hkv < 0)
    return fail(TX_ERR_INVALID, "negative extent");
  if (d.T > INT32_MAX || d.B > INT32_MAX / 2 || d.pages > INT32_MAX || d.table_width > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "extents above 2^31");
  if (d.dtype != TX_F16 && d.dtype != TX_BF16)
    return fail(TX_ERR_UNSUPPORTED, "dtype %d: fp16 and bf16 are implemented", d.dtype);
  if (d.cache_type != d.dtype && d.cache_type != TX_F8E4M3)
    return fail(TX_ERR_UNSUPPORTED, "cache type %d: that of the tokens, or fp8 e4m3",
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

template <class T, class C> void appendKernels(void (*(&k)[2][4])(AppendArgs)) {
  k[0][0] = paged_append_kernel<T, C, 1, false>, k[0][1] = paged_append_kernel<T, C, 2, false>;
  k[0][2] = paged_append_kernel<T, C, 4, false>, k[0][3] = paged_append_kernel<T, C, 8, false>;
  k[1][0] = paged_append_kernel<T, C, 1, true>, k[1][1] = paged_append_kernel<T, C, 2, true>;
  k[1][2] = paged_append_kernel<T, C, 4, true>, k[1][3] = paged_append_kernel<T, C, 8, true>;
}

} // namespace

extern "C" TX_API int tx_paged_append_plan_create(const tx_paged_append_desc *desc,
                                                  tx_paged_append_plan *plan) {
  clearError();
  if (!desc || !plan)
    return fail(TX_ERR_INVALID, "descriptor or plan is NULL");
  const tx_paged_append_desc &d = *desc;
  int rc = checkPaged(d, d.interleaved);
  if (rc != TX_OK)
    return rc;
  if (d.rot_dim < 0 || d.rot_dim > d.head_dim || d.rot_dim % 2 || d.head_dim > 65536)
    return fail(TX_ERR_INVALID, "rot_dim %d of head_dim %d: an even number of its dims", d.rot_dim,
                d.head_dim);
  if (!std::isfinite(d.scale))
    return fail(TX_ERR_INVALID, "scale must be finite");
  rc = checkStrides("q", d.T, d.q_st, d.Hq, d.q_sh, d.head_dim, false);
  if (rc == TX_OK && d.Hq) rc = checkStrides("q_out", d.T, d.o_st, d.Hq, d.o_sh, d.head_dim, true);
  if (rc == TX_OK) rc = checkStrides("k", d.T, d.k_st, d.Hkv, d.k_sh, d.head_dim, false);
  if (rc == TX_OK) rc = checkStrides("v", d.T, d.v_st, d.Hkv, d.v_sh, d.head_dim, false);
  if (rc == TX_OK)
    rc = checkCache("k_cache", d.pages, d.kc_sp, d.page_size, d.kc_st, d.Hkv, d.kc_sh, d.head_dim);
  if (rc == TX_OK)
    rc = checkCache("v_cache", d.pages, d.vc_sp, d.page_size, d.vc_st, d.Hkv, d.vc_sh, d.head_dim);
  if (rc != TX_OK)
    return rc;
  std::memset(plan, 0, sizeof(*plan));
  plan->desc = d;
  const double T = (double)d.T;
  plan->flops = 3.0 * T * (d.Hq + d.Hkv) * d.rot_dim;
  plan->bytes = T * d.head_dim * (4.0 * d.Hq + 2.0 * d.Hkv * (2 + sizeOf(d.cache_type)));
  plan->vec = commonVec(vecOf(8, d.head_dim, d.rot_dim, d.interleaved),
                        {d.Hq ? d.q_st : 0, d.Hq ? d.q_sh : 0, d.Hq ? d.o_st : 0,
                         d.Hq ? d.o_sh : 0, d.k_st, d.k_sh, d.v_st, d.v_sh, d.kc_sp, d.kc_st,
                         d.kc_sh, d.vc_sp, d.vc_st, d.vc_sh});
  const int64_t items = itemsOf(d.head_dim, d.rot_dim, plan->vec, d.interleaved);
  const int64_t heads = (int64_t)d.Hq + 2 * (int64_t)d.Hkv;
  plan->head_lanes = headLanes(d.T, items, heads);
  plan->block_threads = 256;
  const int64_t per = items * plan->head_lanes;
  if (tokenGrid(d.T, per) * 32 > INT32_MAX || per > INT32_MAX / 32 || heads > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "grid above 2^31");
  plan->grid_x = heads == 0 ? 0 : (int32_t)tokenGrid(d.T, per);
  return TX_OK;
}

extern "C" TX_API int tx_paged_append_launch(const tx_paged_append_plan *plan, const void *q,
                                             const void *k, const void *v, void *q_out,
                                             void *k_cache, void *v_cache,
                                             const int32_t *page_table, const int32_t *kv_len,
                                             const int32_t *cu_q, const float *inv_freq,
                                             const float *k_scale, const float *v_scale,
                                             void *stream) {
  clearError();
  if (!plan)
    return fail(TX_ERR_INVALID, "plan is NULL");
  tx_paged_append_plan again;
  const int rc = tx_paged_append_plan_create(&plan->desc, &again);
  if (rc != TX_OK)
    return rc;
  if (std::memcmp(&again, plan, sizeof again) != 0)
    return fail(TX_ERR_INVALID, "the plan does not follow from its descriptor");
  if (plan->grid_x == 0)
    return TX_OK;
  const tx_paged_append_desc &d = plan->desc;
  const bool cached = d.Hkv > 0;
  if ((d.Hq && (!q || !q_out)) || (cached && (!k || !v)) || !kv_len ||
      (cached && d.pages > 0 && (!k_cache || !v_cache)) ||
      (cached && d.table_width > 0 && !page_table) || (d.rot_dim && !inv_freq))
    return fail(TX_ERR_INVALID, "NULL tensor pointer");
  if ((cu_q != nullptr) != (d.ragged != 0))
    return fail(TX_ERR_INVALID, "cu_q must be given exactly when the plan is ragged");
  const int64_t ce = sizeOf(d.cache_type);
  for (const void *p : {static_cast<const void *>(page_table), static_cast<const void *>(kv_len),
                        static_cast<const void *>(cu_q), static_cast<const void *>(inv_freq),
                        static_cast<const void *>(k_scale), static_cast<const void *>(v_scale)})
    if (!aligned(p, 4))
      return fail(TX_ERR_INVALID, "index, frequency and scale arrays must be 4-byte aligned");
  const void *tok[4] = {q, k, v, q_out};
  int vec = plan->vec, lanes = plan->head_lanes;
  bool whole = aligned(k_cache, vec * ce) && aligned(v_cache, vec * ce);
  for (const void *p : tok) {
    if (!aligned(p, 2))
      return fail(TX_ERR_INVALID, "a tensor is not aligned to its elements");
    whole = whole && aligned(p, vec * 2);
  }
  if (!aligned(k_cache, ce) || !aligned(v_cache, ce))
    return fail(TX_ERR_INVALID, "a cache is not aligned to its elements");
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  const int64_t heads = (int64_t)d.Hq + 2 * (int64_t)d.Hkv;
  if (!whole) {
    vec = 1;
    lanes = headLanes(d.T, itemsOf(d.head_dim, d.rot_dim, 1, d.interleaved), heads);
  }
  AppendArgs a;
  a.q = q, a.k = k, a.v = v, a.q_out = q_out;
  a.kc = static_cast<uint8_t *>(k_cache), a.vc = static_cast<uint8_t *>(v_cache);
  a.table = page_table, a.kv_len = kv_len, a.cu_q = cu_q;
  a.inv_freq = inv_freq, a.k_scale = k_scale, a.v_scale = v_scale;
  a.T = d.T, a.pages = k_cache && v_cache ? d.pages : 0;
  a.table_width = page_table ? d.table_width : 0, a.table_s = d.table_s;
  a.q_st = d.q_st, a.q_sh = d.q_sh, a.o_st = d.o_st, a.o_sh = d.o_sh;
  a.k_st = d.k_st, a.k_sh = d.k_sh, a.v_st = d.v_st, a.v_sh = d.v_sh;
  a.kc_sp = d.kc_sp, a.kc_st = d.kc_st, a.kc_sh = d.kc_sh;
  a.vc_sp = d.vc_sp, a.vc_st = d.vc_st, a.vc_sh = d.vc_sh;
  a.B = (int32_t)d.B, a.Hq = d.Hq, a.Hkv = d.Hkv, a.head_dim = d.head_dim, a.rot = d.rot_dim;
  a.items = itemsOf(d.head_dim, d.rot_dim, vec, d.interleaved);
  a.token_threads = a.items * lanes;
  a.head_lanes = lanes, a.page_shift = log2of(d.page_size), a.scale = d.scale;
  void (*fn[2][4])(AppendArgs);
  const bool f8 = d.cache_type == TX_F8E4M3;
  if (d.dtype == TX_F16 && f8)
    appendKernels<_Float16, uint8_t>(fn);
  else if (d.dtype == TX_F16)
    appendKernels<_Float16, _Float16>(fn);
  else if (f8)
    appendKernels<__bf16, uint8_t>(fn);
  else
    appendKernels<__bf16, __bf16>(fn);
  hipLaunchKernelGGL(fn[d.interleaved][log2of(vec)],
                     dim3((uint32_t)tokenGrid(d.T, a.token_threads)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}

// ---------------------------------------------------------------------------
// Attention over the cache
// ---------------------------------------------------------------------------

namespace {

constexpr int64_t kAttnCounters = 65536; // the arrival counters that every workspace begins with

// The dims that a head is computed in.
int attnDims(int head_dim) {
  return head_dim <= 64 ? 64 : head_dim <= 96 ? 96 : head_dim <= 128 ? 128 : 256;
}
// Forms of the kernel, by the rows of a unit: 16, 32 (the waves of a workgroup share out the keys,
// in blocks of 32), 128 (they share the keys, in blocks of 64).
enum { kAttn16 = 0, kAttn32 = 1, kAttn128 = 2 };
constexpr int kSplitBlock = 32;

// Rows of a page that one buffer resource covers: as many as divide a page and the rows
// that a wave loads, with 31-bit offsets.
int runOf(int rows, int page_size, int64_t st, int64_t row_bytes) {
  int run = std::min(rows, page_size);
  while (run > 1 && ((run - 1) * st + row_bytes >= ((int64_t)1 << 31) || st >= ((int64_t)1 << 31)))
    run /= 2;
  return run;
}

} // namespace

extern "C" TX_API int tx_paged_attn_plan_create(const tx_paged_attn_desc *desc,
                                                tx_paged_attn_plan *plan) {
  clearError();
  if (!desc || !plan)
    return fail(TX_ERR_INVALID, "descriptor or plan is NULL");
  const tx_paged_attn_desc &d = *desc;
  int rc = checkPaged(d, d.causal);
  if (rc != TX_OK)
    return rc;
  if (d.T > 0 && (d.Hq < 1 || d.Hkv < 1 || d.Hq % d.Hkv))
    return fail(TX_ERR_INVALID, "%d query heads of %d key heads: a multiple", d.Hq, d.Hkv);
  const int64_t ce = sizeOf(d.cache_type), quantum = 16 / ce;
  if (d.head_dim > 256 || d.head_dim % quantum)
    return fail(TX_ERR_UNSUPPORTED, "head_dim %d: a multiple of %lld up to 256", d.head_dim,
                (long long)quantum);
  if (!std::isfinite(d.sm_scale) || d.sm_scale < 0)
    return fail(TX_ERR_INVALID, "sm_scale must be finite and not negative");
  if (d.window < 0)
    return fail(TX_ERR_INVALID, "window %d", d.window);
  rc = checkStrides("q", d.T, d.q_st, d.Hq, d.q_sh, d.head_dim, false);
  if (rc == TX_OK) rc = checkStrides("o", d.T, d.o_st, d.Hq, d.o_sh, d.head_dim, true);
  if (rc == TX_OK)
    rc = checkCache("k_cache", d.pages, d.k_sp, d.page_size, d.k_st, d.Hkv, d.k_sh, d.head_dim);
  if (rc == TX_OK)
    rc = checkCache("v_cache", d.pages, d.v_sp, d.page_size, d.v_st, d.Hkv, d.v_sh, d.head_dim);
  if (rc != TX_OK)
    return rc;
  if (d.q_st % 8 || d.q_sh % 8 || d.o_st % 8 || d.o_sh % 8)
    return fail(TX_ERR_INVALID, "q and o strides must be multiples of 16 bytes");
  if (d.k_sp % quantum || d.k_st % quantum || d.k_sh % quantum || d.v_sp % quantum ||
      d.v_st % quantum || d.v_sh % quantum)
    return fail(TX_ERR_INVALID, "cache strides must be multiples of 16 bytes");
  if (d.T * (int64_t)(d.Hkv ? d.Hq / d.Hkv : 0) > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "more than 2^31 rows of a kv head");
  std::memset(plan, 0, sizeof(*plan));
  plan->desc = d;
  plan->block_threads = 256;
  if (d.T == 0)
    return TX_OK;
  // The fewer rows a sequence has on average, the less of a unit's matrix and softmax work is
  // for nothing; past a form's rows its units read the same keys again.  16 sequences of 16384 keys,
  // heads of 128: 32 rows each 204 us in the form of 32, 224 in that of 128; 64 rows 374 and 209.  4
  // rows each (32 sequences of up to 16384): 86 in the form of 16, 90 in that of 32.
  const int64_t G = d.Hq / d.Hkv, rows = d.T * G;
  plan->variant = rows <= 16 * d.B ? kAttn16 : rows <= 32 * d.B ? kAttn32 : kAttn128;
  plan->rows = plan->variant == kAttn16 ? 16 : plan->variant == kAttn32 ? 32 : 128;
  const int D = attnDims(d.head_dim);
  const bool f8 = d.cache_type == TX_F8E4M3;
  // workgroups that a CU has place for (by LDS and registers)
  const bool one = D > 128 && !(plan->variant == kAttn16 && f8);
  const int per_cu = one ? 1 : plan->variant == kAttn128 && D == 64 ? 3 : 2;
  // the most steps of work there can be (a step: the keys a workgroup takes at a time)
  const bool split = plan->variant != kAttn128;
  const int step = split ? 4 * kSplitBlock : 64;
  const double units = (double)d.B + (double)d.T * G / plan->rows;
  const double keys = (double)d.table_width * d.page_size;
  const double steps = units * (keys / step + 1 + (split ? kSplitOverhead : kRowsOverhead)) * d.Hkv;
  if (steps > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "more than 2^31 blocks of keys for %lld tokens: fewer a call",
                (long long)d.T);
  plan->units = (int32_t)std::min<double>(256 * per_cu, std::ceil(steps));
  plan->grid_x = plan->units;
  plan->slots = 2 * plan->units;
  plan->workspace_bytes =
      kAttnCounters + (int64_t)plan->slots * plan->rows * (D + 2) * (int64_t)sizeof(float);
  return TX_OK;
}

extern "C" TX_API int tx_paged_attn_launch(const tx_paged_attn_plan *plan, const void *q,
                                           const void *k_cache, const void *v_cache,
                                           const int32_t *page_table, const int32_t *kv_len,
                                           const int32_t *cu_q, const float *k_scale,
                                           const float *v_scale, void *o, float *lse,
                                           void *workspace, size_t workspace_bytes, void *stream) {
  clearError();
  if (!plan)
    return fail(TX_ERR_INVALID, "plan is NULL");
  tx_paged_attn_plan again;
  const int rc = tx_paged_attn_plan_create(&plan->desc, &again);
  if (rc != TX_OK)
    return rc;
  if (std::memcmp(&again, plan, sizeof again) != 0)
    return fail(TX_ERR_INVALID, "the plan does not follow from its descriptor");
  if (plan->grid_x == 0)
    return TX_OK;
  const tx_paged_attn_desc &d = plan->desc;
  if (!q || !o || !kv_len || (d.pages > 0 && (!k_cache || !v_cache)) ||
      (d.table_width > 0 && !page_table))
    return fail(TX_ERR_INVALID, "NULL tensor pointer");
  if ((cu_q != nullptr) != (d.ragged != 0))
    return fail(TX_ERR_INVALID, "cu_q must be given exactly when the plan is ragged");
  if (!aligned(q, 16) || !aligned(o, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(TX_ERR_INVALID, "q, o and the caches must be 16-byte aligned");
  for (const void *p : {static_cast<const void *>(page_table), static_cast<const void *>(kv_len),
                        static_cast<const void *>(cu_q), static_cast<const void *>(k_scale),
                        static_cast<const void *>(v_scale), static_cast<const void *>(lse)})
    if (!aligned(p, 4))
      return fail(TX_ERR_INVALID, "index, scale and lse arrays must be 4-byte aligned");
  if (plan->workspace_bytes > 0 &&
      (!workspace || workspace_bytes < (size_t)plan->workspace_bytes || !aligned(workspace, 256)))
    return fail(TX_ERR_WORKSPACE, "the plan needs %lld bytes of workspace, 256-byte aligned",
                (long long)plan->workspace_bytes);
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  PagedAttnArgs a;
  const bool f8 = d.cache_type == TX_F8E4M3;
  const int64_t ce = f8 ? 1 : 2;
  const int D = attnDims(d.head_dim);
  a.q = q, a.o = o, a.lse = lse;
  a.kc = static_cast<const uint8_t *>(k_cache), a.vc = static_cast<const uint8_t *>(v_cache);
  a.table = page_table, a.kv_len = kv_len, a.cu_q = cu_q;
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.counters = static_cast<uint32_t *>(workspace);
  a.parts = static_cast<uint8_t *>(workspace) + kAttnCounters;
  a.table_width = d.table_width, a.table_s = d.table_s;
  a.most = (int32_t)std::min<int64_t>(d.table_width * d.page_size, INT32_MAX - 127);
  a.q_st = d.q_st, a.q_sh = d.q_sh, a.o_st = d.o_st, a.o_sh = d.o_sh;
  a.k_sp = d.k_sp * ce, a.k_st = d.k_st * ce, a.k_sh = d.k_sh * ce;
  a.v_sp = d.v_sp * ce, a.v_st = d.v_st * ce, a.v_sh = d.v_sh * ce;
  a.pages = (uint32_t)d.pages;
  a.g_mul = a.g_shift = 0;
  if (const int64_t G = d.Hq / d.Hkv; G > 1) { // ceil(2^(31 + s) / G), 2^s >= G
    const int sh = log2of(G);
    a.g_mul = (uint32_t)((((uint64_t)1 << (31 + sh)) + G - 1) / G), a.g_shift = sh - 1;
  }
  a.T = (int32_t)d.T, a.B = (int32_t)d.B, a.G = d.Hq / d.Hkv, a.Hq = d.Hq, a.Hkv = d.Hkv;
  a.head_dim = d.head_dim, a.page_shift = log2of(d.page_size);
  a.causal = d.causal, a.window = d.window;
  const int wave_rows = plan->variant == kAttn128 ? 16 : kSplitBlock;
  a.k_run = runOf(wave_rows, d.page_size, a.k_st, d.head_dim * ce);
  a.v_run = runOf(wave_rows, d.page_size, a.v_st, d.head_dim * ce);
  a.qk_scale = d.sm_scale * 1.44269504f;
  const PagedAttnFn fn =
      (plan->variant == kAttn16 ? kPagedAttnSplit16
       : plan->variant == kAttn32 ? kPagedAttnSplit
                                  : kPagedAttnRows)[D == 64 ? 0 : D == 96 ? 1 : D == 128 ? 2 : 3]
                                       [d.dtype == TX_BF16][f8];
  hipLaunchKernelGGL(fn, dim3(plan->grid_x), dim3(plan->block_threads), 0,
                     static_cast<hipStream_t>(stream), a);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}

// ---------------------------------------------------------------------------
// Pages
// ---------------------------------------------------------------------------

namespace {

int checkPageDesc(const tx_page_desc *d) {
  if (!d)
    return fail(TX_ERR_INVALID, "descriptor is NULL");
  if (d->S < 0 || d->W < 0 || d->P < 0 || d->n < 0)
    return fail(TX_ERR_INVALID, "negative extent");
  // entries are counted in int32
  if (d->P > INT32_MAX || d->W > INT32_MAX || (d->W && d->S > INT32_MAX / d->W) ||
      d->S > INT32_MAX || (d->W && d->n > INT32_MAX / d->W) || d->n > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "extents above 2^31");
  if (!pow2(d->page_size) || d->page_size > 65536)
    return fail(TX_ERR_UNSUPPORTED, "page_size %d: a power of two up to 65536", d->page_size);
  if (d->caches < 0 || d->caches > TX_PAGE_CACHES)
    return fail(TX_ERR_UNSUPPORTED, "%d caches: at most %d a call", d->caches, TX_PAGE_CACHES);
  for (int i = 0; i < d->caches; ++i) {
    if (d->bytes[i] < 0 || d->bytes[i] % 16 || d->stride[i] % 16)
      return fail(TX_ERR_INVALID, "cache %d: pages must be multiples of 16 bytes", i);
    if (d->P > 1 && d->stride[i] < d->bytes[i])
      return fail(TX_ERR_INVALID, "cache %d: pages overlap", i);
  }
  return TX_OK;
}
int checkPages(const tx_page_desc *d, void *const *caches) {
  const int rc = checkPageDesc(d);
  if (rc != TX_OK)
    return rc;
  if (d->caches && !caches)
    return fail(TX_ERR_INVALID, "caches is NULL");
  for (int i = 0; i < d->caches; ++i) {
    if (!caches[i] && d->P > 0 && d->bytes[i] > 0)
      return fail(TX_ERR_INVALID, "cache %d is NULL", i);
    if (!aligned(caches[i], 16))
      return fail(TX_ERR_INVALID, "cache %d is not 16-byte aligned", i);
  }
  return TX_OK;
}

// Whether an array is NULL that a call on books of these extents reads or writes.
bool anyNull(const tx_page_desc &d, std::initializer_list<const void *> of_S,
             std::initializer_list<const void *> of_table, std::initializer_list<const void *> of_P) {
  for (const void *p : of_S)
    if (!p && d.S)
      return true;
  for (const void *p : of_table)
    if (!p && d.S && d.W)
      return true;
  for (const void *p : of_P)
    if (!p && d.P)
      return true;
  return false;
}
BookArgs bookArgs(const tx_page_desc &d, const int32_t *table, const int32_t *len,
                  const int32_t *refs, int32_t *table_out, int32_t *len_out, int32_t *refs_out,
                  int32_t *count, void *workspace) {
  BookArgs a = {};
  a.W = d.W, a.S = (int32_t)d.S, a.P = (int32_t)d.P, a.n = (int32_t)d.n;
  a.page_shift = log2of(d.page_size);
  a.table = table, a.len = len, a.refs = refs;
  a.table_out = table_out, a.len_out = len_out, a.refs_out = refs_out, a.count = count;
  a.table_in_place = table_out == table, a.refs_in_place = refs_out == refs;
  a.src = static_cast<int32_t *>(workspace);
  if (workspace)
    a.dst = a.src + 2 * std::max(d.P, d.n);
  return a;
}

// Workgroups over the table's rows: about 2048 entries (or counts) each; `alone`: one.
int64_t bookGrid(const tx_page_desc &d, bool alone, BookArgs &a) {
  int64_t grid = std::max(cdiv(d.S * d.W, 2048), cdiv(d.P, 4096));
  grid = alone ? 1 : std::min<int64_t>(std::max<int64_t>(grid, 1), 256);
  a.rows = (int32_t)std::min<int64_t>(std::max<int64_t>(cdiv(d.S, grid), 1), kBookRows);
  return grid;
}

int launchCopy(const tx_page_desc &d, void *const *caches, const int32_t *src, const int32_t *dst,
               const int32_t *count, int64_t most, hipStream_t s) {
  PageCopyArgs a;
  int64_t pieces = 0;
  a.src = src, a.dst = dst, a.count = count, a.n = most, a.P = d.P, a.caches = d.caches;
  for (int i = 0; i < d.caches; ++i) {
    a.base[i] = static_cast<uint8_t *>(caches[i]);
    a.stride[i] = d.stride[i], a.bytes[i] = d.bytes[i];
    pieces = std::max(pieces, cdiv(d.bytes[i], 16384));
  }
  if (d.caches == 0 || most == 0 || pieces == 0)
    return TX_OK;
  const int64_t per = std::max<int64_t>(1, cdiv(2048, d.caches));
  hipLaunchKernelGGL(page_copy_kernel, dim3((uint32_t)std::min(per, most * pieces), d.caches),
                     dim3(256), 0, s, a);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}

} // namespace

extern "C" TX_API int tx_page_workspace(const tx_page_desc *desc, int64_t *bytes) {
  clearError();
  const int rc = checkPageDesc(desc);
  if (rc != TX_OK)
    return rc;
  if (!bytes)
    return fail(TX_ERR_INVALID, "bytes is NULL");
  // lists of pages to copy (a page and its place each, and the places found), and the bits of
  // page_compact where they do not fit LDS
  *bytes = 12 * std::max(desc->P, desc->n) + 8 + 12 * (cdiv(desc->P, 64) + 1);
  return TX_OK;
}

extern "C" TX_API int tx_page_copy(const tx_page_desc *desc, void *const *caches,
                                   const int32_t *src, const int32_t *dst, void *stream) {
  clearError();
  const int rc = checkPages(desc, caches);
  if (rc != TX_OK)
    return rc;
  if (desc->n == 0 || desc->caches == 0)
    return TX_OK;
  if (!src || !dst)
    return fail(TX_ERR_INVALID, "src or dst is NULL");
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  return launchCopy(*desc, caches, src, dst, nullptr, desc->n, static_cast<hipStream_t>(stream));
}

extern "C" TX_API int tx_page_reserve(const tx_page_desc *desc, const int32_t *page_table,
                                      const int32_t *kv_len, const int32_t *refs,
                                      const int32_t *new_len, int32_t *table_out, int32_t *len_out,
                                      int32_t *refs_out, int32_t *missing, void *workspace,
                                      void *stream) {
  clearError();
  const int rc = checkPageDesc(desc);
  if (rc != TX_OK)
    return rc;
  if (anyNull(*desc, {kv_len, new_len, len_out}, {page_table, table_out}, {refs, refs_out}))
    return fail(TX_ERR_INVALID, "NULL array");
  if (!missing || !workspace)
    return fail(TX_ERR_INVALID, "missing or workspace is NULL");
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  BookArgs a = bookArgs(*desc, page_table, kv_len, refs, table_out, len_out, refs_out, missing,
                        workspace);
  a.new_len = new_len;
  const bool alone = refs_out == refs || len_out == kv_len || len_out == new_len;
  const int64_t grid = bookGrid(*desc, alone, a);
  hipLaunchKernelGGL(page_reserve_kernel, dim3((uint32_t)grid), dim3(kBookThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}

extern "C" TX_API int tx_page_fork(const tx_page_desc *desc, void *const *caches,
                                   const int32_t *page_table, const int32_t *kv_len,
                                   const int32_t *refs, const int32_t *parent,
                                   const int32_t *child, int32_t *table_out, int32_t *len_out,
                                   int32_t *refs_out, int32_t *missing, void *workspace,
                                   void *stream) {
  clearError();
  const int rc = checkPages(desc, caches);
  if (rc != TX_OK)
    return rc;
  if (anyNull(*desc, {kv_len, len_out}, {page_table, table_out}, {refs, refs_out}))
    return fail(TX_ERR_INVALID, "NULL array");
  if (desc->n && (!parent || !child))
    return fail(TX_ERR_INVALID, "parent or child is NULL");
  if (!missing || !workspace)
    return fail(TX_ERR_INVALID, "missing or workspace is NULL");
  if (!aligned(workspace, 8))
    return fail(TX_ERR_WORKSPACE, "workspace must be 8-byte aligned");
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  hipStream_t s = static_cast<hipStream_t>(stream);
  BookArgs a = bookArgs(*desc, page_table, kv_len, refs, table_out, len_out, refs_out, missing,
                        workspace);
  a.parent = parent, a.child = child;
  // one for the children, others for the rows to copy
  const int64_t grid = a.table_in_place && len_out == kv_len ? 1 : 1 + bookGrid(*desc, false, a);
  hipLaunchKernelGGL(page_fork_kernel, dim3((uint32_t)grid), dim3(kBookThreads), 0, s, a);
  TX_HIP_CHECK(hipGetLastError());
  return launchCopy(*desc, caches, a.src, a.dst, nullptr, desc->n, s);
}

extern "C" TX_API int tx_page_free(const tx_page_desc *desc, const int32_t *page_table,
                                   const int32_t *kv_len, const int32_t *refs, const uint8_t *drop,
                                   int32_t *table_out, int32_t *len_out, int32_t *refs_out,
                                   void *stream) {
  clearError();
  const int rc = checkPageDesc(desc);
  if (rc != TX_OK)
    return rc;
  if (anyNull(*desc, {kv_len, drop, len_out}, {page_table, table_out}, {refs, refs_out}))
    return fail(TX_ERR_INVALID, "NULL array");
  if (desc->S == 0)
    if (desc->P == 0 || refs_out == refs)
      return TX_OK;
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  BookArgs a = bookArgs(*desc, page_table, kv_len, refs, table_out, len_out, refs_out, nullptr,
                        nullptr);
  a.drop = drop;
  hipStream_t s = static_cast<hipStream_t>(stream);
  // One launch while a thread has few entries of the table; past it, or in place, a copy of the
  // counts and atomics on them.
  const bool apart = !a.table_in_place && len_out != kv_len;
  if (apart && desc->P > 0 && desc->P <= 256 * kFreePages && desc->S * desc->W > 0 &&
      desc->S * desc->W <= kFreeEntries) {
    hipLaunchKernelGGL(page_free_small_kernel, dim3((uint32_t)cdiv(desc->P, kFreePages)),
                       dim3(kBookThreads), 0, s, a);
    TX_HIP_CHECK(hipGetLastError());
    return TX_OK;
  }
  if (!a.refs_in_place && desc->P > 0) {
    hipLaunchKernelGGL(book_copy_kernel, dim3((uint32_t)std::min<int64_t>(cdiv(desc->P, 256), 1024)),
                       dim3(256), 0, s, refs_out, refs, desc->P);
    TX_HIP_CHECK(hipGetLastError());
  }
  if (desc->S == 0)
    return TX_OK;
  // a row's threads: 64 .. 512 by its length
  int64_t tw = 64;
  while (tw < desc->W && tw < kBookThreads)
    tw *= 2;
  const int64_t grid = std::min<int64_t>(cdiv(desc->S, kBookThreads / tw), 1024);
  hipLaunchKernelGGL(page_free_kernel, dim3((uint32_t)grid), dim3(kBookThreads), 0, s, a);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}

extern "C" TX_API int tx_page_compact(const tx_page_desc *desc, void *const *caches,
                                      const int32_t *page_table, const int32_t *refs,
                                      int32_t *table_out, int32_t *refs_out, int32_t *moved,
                                      void *workspace, void *stream) {
  clearError();
  const int rc = checkPages(desc, caches);
  if (rc != TX_OK)
    return rc;
  if (anyNull(*desc, {}, {page_table, table_out}, {refs, refs_out}))
    return fail(TX_ERR_INVALID, "NULL array");
  if (!moved || !workspace)
    return fail(TX_ERR_INVALID, "moved or workspace is NULL");
  if (!aligned(workspace, 8))
    return fail(TX_ERR_WORKSPACE, "workspace must be 8-byte aligned");
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  hipStream_t s = static_cast<hipStream_t>(stream);
  BookArgs a = bookArgs(*desc, page_table, nullptr, refs, table_out, nullptr, refs_out, moved,
                        workspace);
  const bool in_lds = cdiv(desc->P, 64) <= kBookMasks;
  if (!in_lds)
    a.masks = reinterpret_cast<uint64_t *>(
        static_cast<uint8_t *>(workspace) + (12 * std::max(desc->P, desc->n) + 7) / 8 * 8);
  const int64_t grid = bookGrid(*desc, a.refs_in_place || !in_lds, a);
  hipLaunchKernelGGL(page_compact_kernel, dim3((uint32_t)grid), dim3(kBookThreads), 0, s, a);
  TX_HIP_CHECK(hipGetLastError());
  return launchCopy(*desc, caches, a.src, a.dst, moved, desc->P, s);
}
