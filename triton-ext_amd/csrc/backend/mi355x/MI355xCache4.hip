// Launch layer of the paged cache held in 4 bits, and of reading any paged cache back
// (tx_cache4.h).

#include "cache_host.h"
#include "cache4_rows.h"
#include "paged_attn4.h"
#include "triton_ext/tx_cache4.h"

using namespace txk;

namespace txk {
typedef void (*Paged4AttnFn)(Paged4Args);
// [16, 32 rows][64, 96, 128, 256 dims][bf16][e4m3 scales] (kernels_paged4_*.hip)
extern const Paged4AttnFn kPaged4Split[2][4][2][2], kPaged4Rows[4][2][2];
} // namespace txk

namespace {

// The strides of block scales; written: no two may share a byte.
int checkScales(const tx_block_scales &s, int64_t pages, int64_t page_size, int64_t Hkv, int64_t head_dim,
                bool written) {
  if (s.mode != TX_SCALE_MX32 && s.mode != TX_SCALE_NV16)
    return fail(TX_ERR_UNSUPPORTED, "block scales of mode %d: TX_SCALE_MX32 or TX_SCALE_NV16", s.mode);
  if (s.reserved)
    return fail(TX_ERR_INVALID, "reserved must be 0");
  const int64_t blocks = head_dim / (s.mode == TX_SCALE_MX32 ? 32 : 16);
  const int64_t st[2][4] = {{s.k_sp, s.k_st, s.k_sh, s.k_sb}, {s.v_sp, s.v_st, s.v_sh, s.v_sb}};
  const int64_t n[4] = {pages, page_size, Hkv, blocks};
  for (const auto &x : st) {
    int order[4] = {0, 1, 2, 3};
    std::sort(order, order + 4, [&](int a, int b) { return x[a] < x[b]; });
    int64_t span = 1; // bytes from the first to past the last scale so far
    for (int i : order) {
      if (x[i] < 0)
        return fail(TX_ERR_INVALID, "block scales: negative stride");
      if (n[i] < 2)
        continue;
      if (x[i] > ((int64_t)1 << 46) / n[i])
        return fail(TX_ERR_UNSUPPORTED, "block scales: strides above 2^46");
      if (written && x[i] < span)
        return fail(TX_ERR_INVALID, "block scales: scales that overlap");
      span += (n[i] - 1) * x[i];
    }
  }
  return TX_OK;
}

// A cache of codes: rows of head_dim / 2 bytes, strides multiples of 16.
int checkCodes(const char *name, int64_t pages, int64_t sp, int64_t page_size, int64_t st, int64_t Hkv,
               int64_t sh, int64_t head_dim) {
  const int rc = checkCache(name, pages, sp, page_size, st, Hkv, sh, head_dim / 2);
  if (rc != TX_OK)
    return rc;
  if (sp % 16 || st % 16 || sh % 16)
    return fail(TX_ERR_INVALID, "%s: strides must be multiples of 16 bytes", name);
  return TX_OK;
}

BlockScales scalesOf(const void *p, int64_t sp, int64_t st, int64_t sh, int64_t sb) {
  return BlockScales{static_cast<uint8_t *>(const_cast<void *>(p)), sp, st, sh, sb};
}

template <class T, bool NV> void append4Kernels(void (*(&k)[3][2])(Append4Args)) {
  k[0][0] = paged_append4_kernel<T, NV, kRunAlone, false>, k[0][1] = paged_append4_kernel<T, NV, kRunAlone, true>;
  k[1][0] = paged_append4_kernel<T, NV, kRunHalves, false>, k[1][1] = paged_append4_kernel<T, NV, kRunHalves, true>;
  k[2][0] = paged_append4_kernel<T, NV, kRunPairs, false>, k[2][1] = paged_append4_kernel<T, NV, kRunPairs, true>;
}

// How a thread has a head's dims (cache4_rows.h): halves where blocks end within them.
int runOfAppend(const tx_paged_append_desc &d, int32_t mode) {
  const int two = mode == TX_SCALE_MX32 ? 64 : 32;
  if (d.interleaved && d.rot_dim)
    return kRunPairs;
  return d.rot_dim % two == 0 && (d.head_dim - d.rot_dim) % two == 0 ? kRunHalves : kRunAlone;
}

} // namespace

// ---------------------------------------------------------------------------
// New tokens into the cache
// ---------------------------------------------------------------------------

extern "C" TX_API int tx_paged_append4_plan_create(const tx_paged_append4_desc *desc,
                                                   tx_paged_append4_plan *plan) {
  clearError();
  if (!desc || !plan)
    return fail(TX_ERR_INVALID, "descriptor or plan is NULL");
  const tx_paged_append_desc &d = desc->c;
  int rc = checkPaged(d, d.interleaved, true);
  if (rc != TX_OK)
    return rc;
  if (d.head_dim % 32 || d.head_dim > 65536)
    return fail(TX_ERR_UNSUPPORTED, "head_dim %d: a multiple of 32", d.head_dim);
  if (d.rot_dim < 0 || d.rot_dim > d.head_dim || d.rot_dim % 2)
    return fail(TX_ERR_INVALID, "rot_dim %d of head_dim %d: an even number of its dims", d.rot_dim,
                d.head_dim);
  if (!std::isfinite(d.scale))
    return fail(TX_ERR_INVALID, "scale must be finite");
  rc = checkStrides("q", d.T, d.q_st, d.Hq, d.q_sh, d.head_dim, false);
  if (rc == TX_OK && d.Hq) rc = checkStrides("q_out", d.T, d.o_st, d.Hq, d.o_sh, d.head_dim, true);
  if (rc == TX_OK) rc = checkStrides("k", d.T, d.k_st, d.Hkv, d.k_sh, d.head_dim, false);
  if (rc == TX_OK) rc = checkStrides("v", d.T, d.v_st, d.Hkv, d.v_sh, d.head_dim, false);
  if (rc == TX_OK)
    rc = checkCodes("k_cache", d.pages, d.kc_sp, d.page_size, d.kc_st, d.Hkv, d.kc_sh, d.head_dim);
  if (rc == TX_OK)
    rc = checkCodes("v_cache", d.pages, d.vc_sp, d.page_size, d.vc_st, d.Hkv, d.vc_sh, d.head_dim);
  if (rc == TX_OK)
    rc = checkScales(desc->s, d.pages, d.page_size, d.Hkv, d.head_dim, true);
  if (rc != TX_OK)
    return rc;
  std::memset(plan, 0, sizeof(*plan));
  plan->desc = *desc;
  const double T = (double)d.T;
  plan->flops = 3.0 * T * (d.Hq + d.Hkv) * d.rot_dim;
  plan->bytes = T * d.head_dim *
                (4.0 * d.Hq + 2.0 * d.Hkv * (2.5 + 1.0 / (desc->s.mode == TX_SCALE_MX32 ? 32 : 16)));
  plan->whole = commonVec(8, {d.Hq ? d.q_st : 0, d.Hq ? d.q_sh : 0, d.Hq ? d.o_st : 0, d.Hq ? d.o_sh : 0,
                              d.k_st, d.k_sh, d.v_st, d.v_sh}) == 8 &&
                (d.interleaved || d.rot_dim % 16 == 0);
  plan->run = runOfAppend(d, desc->s.mode);
  const int64_t items = d.head_dim / (plan->run == kRunHalves ? 16 : 8), heads = (int64_t)d.Hq + 2 * (int64_t)d.Hkv;
  plan->head_lanes = headLanes(d.T, items, heads);
  plan->block_threads = 256;
  const int64_t per = items * plan->head_lanes;
  if (tokenGrid(d.T, per) > INT32_MAX || per > INT32_MAX || heads > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "grid above 2^31");
  plan->grid_x = heads == 0 ? 0 : (int32_t)tokenGrid(d.T, per);
  return TX_OK;
}

extern "C" TX_API int tx_paged_append4_launch(const tx_paged_append4_plan *plan, const void *q,
                                              const void *k, const void *v, void *q_out, void *k_cache,
                                              void *v_cache, void *k_block_scale, void *v_block_scale,
                                              const int32_t *page_table, const int32_t *kv_len,
                                              const int32_t *cu_q, const float *inv_freq,
                                              const float *k_scale, const float *v_scale, void *stream) {
  clearError();
  if (!plan)
    return fail(TX_ERR_INVALID, "plan is NULL");
  tx_paged_append4_plan again;
  const int rc = tx_paged_append4_plan_create(&plan->desc, &again);
  if (rc != TX_OK)
    return rc;
  if (std::memcmp(&again, plan, sizeof again) != 0)
    return fail(TX_ERR_INVALID, "the plan does not follow from its descriptor");
  if (plan->grid_x == 0)
    return TX_OK;
  const tx_paged_append_desc &d = plan->desc.c;
  const tx_block_scales &s = plan->desc.s;
  const bool cached = d.Hkv > 0;
  if ((d.Hq && (!q || !q_out)) || (cached && (!k || !v)) || !kv_len ||
      (cached && d.pages > 0 && (!k_cache || !v_cache || !k_block_scale || !v_block_scale)) ||
      (cached && d.table_width > 0 && !page_table) || (d.rot_dim && !inv_freq))
    return fail(TX_ERR_INVALID, "NULL tensor pointer");
  if ((cu_q != nullptr) != (d.ragged != 0))
    return fail(TX_ERR_INVALID, "cu_q must be given exactly when the plan is ragged");
  for (const void *p : {static_cast<const void *>(page_table), static_cast<const void *>(kv_len),
                        static_cast<const void *>(cu_q), static_cast<const void *>(inv_freq),
                        static_cast<const void *>(k_scale), static_cast<const void *>(v_scale)})
    if (!aligned(p, 4))
      return fail(TX_ERR_INVALID, "index, frequency and scale arrays must be 4-byte aligned");
  bool whole = plan->whole;
  for (const void *p : {q, k, v, static_cast<const void *>(q_out)}) {
    if (!aligned(p, 2))
      return fail(TX_ERR_INVALID, "a tensor is not aligned to its elements");
    whole = whole && aligned(p, 16);
  }
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(TX_ERR_INVALID, "the caches must be 16-byte aligned");
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  Append4Args g;
  AppendArgs &a = g.a;
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
  a.items = d.head_dim / (plan->run == kRunHalves ? 16 : 8);
  a.head_lanes = plan->head_lanes, a.token_threads = a.items * plan->head_lanes;
  a.page_shift = log2of(d.page_size), a.scale = d.scale;
  g.ks = scalesOf(k_block_scale, s.k_sp, s.k_st, s.k_sh, s.k_sb);
  g.vs = scalesOf(v_block_scale, s.v_sp, s.v_st, s.v_sh, s.v_sb);
  // values of the type at the ends: 6 * 2^hi is one, 0.5 * 2^lo is exact
  g.lo = d.dtype == TX_F16 ? -23 : -125, g.hi = d.dtype == TX_F16 ? 13 : 125;
  void (*fn[3][2])(Append4Args);
  const bool nv = s.mode == TX_SCALE_NV16;
  if (d.dtype == TX_F16 && nv)
    append4Kernels<_Float16, true>(fn);
  else if (d.dtype == TX_F16)
    append4Kernels<_Float16, false>(fn);
  else if (nv)
    append4Kernels<__bf16, true>(fn);
  else
    append4Kernels<__bf16, false>(fn);
  hipLaunchKernelGGL(fn[plan->run][whole], dim3((uint32_t)plan->grid_x), dim3(256), 0,
                     static_cast<hipStream_t>(stream), g);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}

// ---------------------------------------------------------------------------
// Tokens out of a cache
// ---------------------------------------------------------------------------

namespace {

typedef void (*ReadFn)(ReadArgs);

template <class C, class O> ReadFn readKernel(int vec, bool whole) {
  if constexpr (!IsE2m1<C>::value)
    if (vec == 1)
      return paged_read_kernel<C, O, 1, false>;
  return whole ? paged_read_kernel<C, O, 8, true> : paged_read_kernel<C, O, 8, false>;
}
template <class C> ReadFn readKernel(int32_t out, int vec, bool whole) {
  return out == TX_F32   ? readKernel<C, float>(vec, whole)
         : out == TX_F16 ? readKernel<C, _Float16>(vec, whole)
                         : readKernel<C, __bf16>(vec, whole);
}

} // namespace

extern "C" TX_API int tx_paged_read_plan_create(const tx_paged_read_desc *desc, tx_paged_read_plan *plan) {
  clearError();
  if (!desc || !plan)
    return fail(TX_ERR_INVALID, "descriptor or plan is NULL");
  const tx_paged_read_desc &d = *desc;
  if (d.out_type != TX_F32 && d.out_type != TX_F16 && d.out_type != TX_BF16)
    return fail(TX_ERR_UNSUPPORTED, "out_type %d: fp32, fp16 and bf16 are implemented", d.out_type);
  const bool packed = d.cache_type == TX_F4E2M1;
  if (!packed && d.cache_type != TX_F16 && d.cache_type != TX_BF16 && d.cache_type != TX_F8E4M3)
    return fail(TX_ERR_UNSUPPORTED, "cache type %d: fp16, bf16, fp8 e4m3 or e2m1", d.cache_type);
  // (what the caches of new tokens are asked, of T tokens of the cache's own type)
  tx_paged_append_desc c = {};
  c.T = d.T, c.B = d.B, c.pages = d.pages, c.table_width = d.table_width, c.Hkv = d.Hkv;
  c.head_dim = d.head_dim, c.page_size = d.page_size, c.ragged = d.ragged, c.table_s = d.table_s;
  c.cache_type = d.cache_type, c.dtype = d.cache_type == TX_F16 ? TX_F16 : TX_BF16;
  int rc = checkPaged(c, 0, packed);
  if (rc != TX_OK)
    return rc;
  if (d.head_dim > 65536 || (packed && d.head_dim % 32))
    return fail(TX_ERR_UNSUPPORTED, "head_dim %d: up to 65536, of e2m1 a multiple of 32", d.head_dim);
  rc = checkStrides("k", d.T, d.k_st, d.Hkv, d.k_sh, d.head_dim, true);
  if (rc == TX_OK) rc = checkStrides("v", d.T, d.v_st, d.Hkv, d.v_sh, d.head_dim, true);
  if (rc != TX_OK)
    return rc;
  if (packed) {
    rc = checkCodes("k_cache", d.pages, d.kc_sp, d.page_size, d.kc_st, d.Hkv, d.kc_sh, d.head_dim);
    if (rc == TX_OK)
      rc = checkCodes("v_cache", d.pages, d.vc_sp, d.page_size, d.vc_st, d.Hkv, d.vc_sh, d.head_dim);
    if (rc == TX_OK)
      rc = checkScales(d.s, d.pages, d.page_size, d.Hkv, d.head_dim, false);
  } else {
    rc = checkCache("k_cache", d.pages, d.kc_sp, d.page_size, d.kc_st, d.Hkv, d.kc_sh, d.head_dim);
    if (rc == TX_OK)
      rc = checkCache("v_cache", d.pages, d.vc_sp, d.page_size, d.vc_st, d.Hkv, d.vc_sh, d.head_dim);
    const tx_block_scales none = {};
    if (rc == TX_OK && std::memcmp(&none, &d.s, sizeof none) != 0)
      return fail(TX_ERR_INVALID, "block scales are of e2m1 caches");
  }
  if (rc != TX_OK)
    return rc;
  std::memset(plan, 0, sizeof(*plan));
  plan->desc = d;
  const double held = packed ? 0.5 + 1.0 / (d.s.mode == TX_SCALE_MX32 ? 32 : 16) : (double)sizeOf(d.cache_type);
  plan->bytes = 2.0 * d.T * d.Hkv * d.head_dim * (held + sizeOf(d.out_type));
  plan->vec = packed || commonVec(8, {d.head_dim, d.kc_sp, d.kc_st, d.kc_sh, d.vc_sp, d.vc_st, d.vc_sh, d.k_st,
                                      d.k_sh, d.v_st, d.v_sh}) == 8
                  ? 8
                  : 1;
  const int64_t items = d.head_dim / plan->vec, heads = 2 * (int64_t)d.Hkv;
  plan->head_lanes = headLanes(d.T, items, heads);
  plan->block_threads = 256;
  const int64_t per = items * plan->head_lanes;
  // (a base that is less aligned than vec runs at vec 1, with 8 times the threads at most)
  if (tokenGrid(d.T, per) * 16 > INT32_MAX || per > INT32_MAX / 16 || heads > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "grid above 2^31");
  plan->grid_x = heads == 0 ? 0 : (int32_t)tokenGrid(d.T, per);
  return TX_OK;
}

extern "C" TX_API int tx_paged_read_launch(const tx_paged_read_plan *plan, const void *k_cache,
                                           const void *v_cache, const void *k_block_scale,
                                           const void *v_block_scale, const int32_t *page_table,
                                           const int32_t *kv_len, const int32_t *cu_q,
                                           const float *k_scale, const float *v_scale, void *k, void *v,
                                           void *stream) {
  clearError();
  if (!plan)
    return fail(TX_ERR_INVALID, "plan is NULL");
  tx_paged_read_plan again;
  const int rc = tx_paged_read_plan_create(&plan->desc, &again);
  if (rc != TX_OK)
    return rc;
  if (std::memcmp(&again, plan, sizeof again) != 0)
    return fail(TX_ERR_INVALID, "the plan does not follow from its descriptor");
  if (plan->grid_x == 0)
    return TX_OK;
  const tx_paged_read_desc &d = plan->desc;
  const bool packed = d.cache_type == TX_F4E2M1;
  if (!k || !v || !kv_len ||
      (d.pages > 0 && (!k_cache || !v_cache || (packed && (!k_block_scale || !v_block_scale)))) ||
      (d.table_width > 0 && !page_table))
    return fail(TX_ERR_INVALID, "NULL tensor pointer");
  if ((cu_q != nullptr) != (d.ragged != 0))
    return fail(TX_ERR_INVALID, "cu_q must be given exactly when the plan is ragged");
  for (const void *p : {static_cast<const void *>(page_table), static_cast<const void *>(kv_len),
                        static_cast<const void *>(cu_q), static_cast<const void *>(k_scale),
                        static_cast<const void *>(v_scale)})
    if (!aligned(p, 4))
      return fail(TX_ERR_INVALID, "index and scale arrays must be 4-byte aligned");
  const int64_t ce = packed ? 16 : sizeOf(d.cache_type), oe = sizeOf(d.out_type);
  if (!aligned(k_cache, ce) || !aligned(v_cache, ce) || !aligned(k, oe) || !aligned(v, oe))
    return fail(TX_ERR_INVALID, "a tensor is not aligned to its elements (e2m1: to 16 bytes)");
  if (!tx_device_available())
    return fail(TX_ERR_NO_DEVICE, "no gfx950 device visible");
  int vec = plan->vec, lanes = plan->head_lanes;
  const bool out16 = commonVec(8, {d.k_st, d.k_sh, d.v_st, d.v_sh}) == 8 && aligned(k, 16) && aligned(v, 16);
  if (!packed && (!out16 || !aligned(k_cache, 8 * ce) || !aligned(v_cache, 8 * ce)) && vec == 8) {
    vec = 1;
    lanes = headLanes(d.T, d.head_dim, 2 * (int64_t)d.Hkv);
  }
  ReadArgs a;
  a.kc = static_cast<const uint8_t *>(k_cache), a.vc = static_cast<const uint8_t *>(v_cache);
  a.ks = scalesOf(k_block_scale, d.s.k_sp, d.s.k_st, d.s.k_sh, d.s.k_sb);
  a.vs = scalesOf(v_block_scale, d.s.v_sp, d.s.v_st, d.s.v_sh, d.s.v_sb);
  a.table = page_table, a.kv_len = kv_len, a.cu_q = cu_q, a.k_scale = k_scale, a.v_scale = v_scale;
  a.k = k, a.v = v;
  a.T = d.T, a.pages = d.pages, a.table_width = page_table ? d.table_width : 0, a.table_s = d.table_s;
  const int64_t unit = packed ? 1 : ce;
  a.kc_sp = d.kc_sp * unit, a.kc_st = d.kc_st * unit, a.kc_sh = d.kc_sh * unit;
  a.vc_sp = d.vc_sp * unit, a.vc_st = d.vc_st * unit, a.vc_sh = d.vc_sh * unit;
  a.k_st = d.k_st, a.k_sh = d.k_sh, a.v_st = d.v_st, a.v_sh = d.v_sh;
  a.B = (int32_t)d.B, a.Hkv = d.Hkv, a.head_dim = d.head_dim;
  a.items = d.head_dim / vec, a.head_lanes = lanes, a.token_threads = a.items * lanes;
  a.page_shift = log2of(d.page_size);
  const ReadFn fn = d.cache_type == TX_F16      ? readKernel<_Float16>(d.out_type, vec, out16)
                    : d.cache_type == TX_BF16   ? readKernel<__bf16>(d.out_type, vec, out16)
                    : d.cache_type == TX_F8E4M3 ? readKernel<E4m3>(d.out_type, vec, out16)
                    : d.s.mode == TX_SCALE_MX32 ? readKernel<E2m1<false>>(d.out_type, vec, out16)
                                                : readKernel<E2m1<true>>(d.out_type, vec, out16);
  hipLaunchKernelGGL(fn, dim3((uint32_t)tokenGrid(d.T, a.token_threads)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}

// ---------------------------------------------------------------------------
// Attention over the cache
// ---------------------------------------------------------------------------

extern "C" TX_API int tx_paged_attn4_plan_create(const tx_paged_attn4_desc *desc, tx_paged_attn4_plan *plan) {
  clearError();
  if (!desc || !plan)
    return fail(TX_ERR_INVALID, "descriptor or plan is NULL");
  const tx_paged_attn_desc &d = desc->c;
  int rc = checkPaged(d, d.causal, true);
  if (rc != TX_OK)
    return rc;
  if (d.T > 0 && (d.Hq < 1 || d.Hkv < 1 || d.Hq % d.Hkv))
    return fail(TX_ERR_INVALID, "%d query heads of %d key heads: a multiple", d.Hq, d.Hkv);
  if (d.head_dim > 256 || d.head_dim % 32)
    return fail(TX_ERR_UNSUPPORTED, "head_dim %d: a multiple of 32 up to 256", d.head_dim);
  if (!std::isfinite(d.sm_scale) || d.sm_scale < 0)
    return fail(TX_ERR_INVALID, "sm_scale must be finite and not negative");
  if (d.window < 0)
    return fail(TX_ERR_INVALID, "window %d", d.window);
  rc = checkStrides("q", d.T, d.q_st, d.Hq, d.q_sh, d.head_dim, false);
  if (rc == TX_OK) rc = checkStrides("o", d.T, d.o_st, d.Hq, d.o_sh, d.head_dim, true);
  if (rc == TX_OK)
    rc = checkCodes("k_cache", d.pages, d.k_sp, d.page_size, d.k_st, d.Hkv, d.k_sh, d.head_dim);
  if (rc == TX_OK)
    rc = checkCodes("v_cache", d.pages, d.v_sp, d.page_size, d.v_st, d.Hkv, d.v_sh, d.head_dim);
  if (rc == TX_OK)
    rc = checkScales(desc->s, d.pages, d.page_size, d.Hkv, d.head_dim, false);
  if (rc != TX_OK)
    return rc;
  if (d.q_st % 8 || d.q_sh % 8 || d.o_st % 8 || d.o_sh % 8)
    return fail(TX_ERR_INVALID, "q and o strides must be multiples of 16 bytes");
  // (the kernels' offsets from one of 16 tokens have 32 bits)
  const tx_block_scales &s = desc->s;
  const int64_t blocks = d.head_dim / (s.mode == TX_SCALE_MX32 ? 32 : 16), far = (int64_t)1 << 26;
  if (d.page_size > 1 && (d.k_st >= far || d.v_st >= far || s.k_st >= far || s.v_st >= far))
    return fail(TX_ERR_UNSUPPORTED, "tokens of a page 2^26 bytes apart");
  if ((blocks - 1) * s.k_sb >= ((int64_t)1 << 31) || (blocks - 1) * s.v_sb >= ((int64_t)1 << 31))
    return fail(TX_ERR_UNSUPPORTED, "scales of a head 2^31 bytes apart");
  if (d.T * (int64_t)(d.Hkv ? d.Hq / d.Hkv : 0) > INT32_MAX)
    return fail(TX_ERR_UNSUPPORTED, "more than 2^31 rows of a kv head");
  std::memset(plan, 0, sizeof(*plan));
  plan->desc = *desc;
  plan->block_threads = 256;
  if (d.T == 0)
    return TX_OK;
  // The fewer rows a sequence has on average, the less of a unit's matrix and softmax work is for
  // nothing; past a form's rows its units convert the same keys again, which the form of 128 does once
  // for all of its waves.  16 sequences of 16384 keys, heads of 128: 16 rows each 68 us in the form of 16,
  // 82 in that of 32; 32 rows 89, and 146 in that of 128; 64 rows 160 and 175.  Heads of 64: 32 rows 67
  // and 90, 64 rows 118 and 106.  8 sequences, heads of 256: 64 rows 131 and 170.  The average decides for all
  // of a call: one chunk of 2048 tokens beside 47 single ones, 8192 keys each, 32 heads of 128 over 8, takes 538
  // us, and 397 in two calls, the chunk by itself.
  const int D = attnDims(d.head_dim);
  const int64_t G = d.Hq / d.Hkv, rows = d.T * G;
  plan->variant = rows <= 16 * d.B ? 0 : rows <= (D > 64 ? 64 : 32) * d.B ? 1 : 2;
  plan->rows = plan->variant == 0 ? 16 : plan->variant == 1 ? 32 : 128;
  // workgroups that a CU has place for (by LDS and registers)
  const int per_cu = plan->variant == 0 ? 2 : D > 128 ? 1 : plan->variant == 2 && D == 64 ? 3 : 2;
  // the most steps of work there can be (a step: the keys a workgroup takes at a time)
  const bool split = plan->variant != 2;
  const int step = split ? 128 : 64;
  const double units = (double)d.B + (double)d.T * G / plan->rows;
  const double keys = (double)d.table_width * d.page_size;
  const double steps = units * (keys / step + 1 + (split ? kSplit4Overhead : kRows4Overhead)) * d.Hkv;
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

extern "C" TX_API int tx_paged_attn4_launch(const tx_paged_attn4_plan *plan, const void *q,
                                            const void *k_cache, const void *v_cache,
                                            const void *k_block_scale, const void *v_block_scale,
                                            const int32_t *page_table, const int32_t *kv_len,
                                            const int32_t *cu_q, const float *k_scale,
                                            const float *v_scale, void *o, float *lse, void *workspace,
                                            size_t workspace_bytes, void *stream) {
  clearError();
  if (!plan)
    return fail(TX_ERR_INVALID, "plan is NULL");
  tx_paged_attn4_plan again;
  const int rc = tx_paged_attn4_plan_create(&plan->desc, &again);
  if (rc != TX_OK)
    return rc;
  if (std::memcmp(&again, plan, sizeof again) != 0)
    return fail(TX_ERR_INVALID, "the plan does not follow from its descriptor");
  if (plan->grid_x == 0)
    return TX_OK;
  const tx_paged_attn_desc &d = plan->desc.c;
  const tx_block_scales &s = plan->desc.s;
  if (!q || !o || !kv_len ||
      (d.pages > 0 && (!k_cache || !v_cache || !k_block_scale || !v_block_scale)) ||
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
  Paged4Args g;
  PagedAttnArgs &a = g.a;
  a.q = q, a.o = o, a.lse = lse;
  a.kc = static_cast<const uint8_t *>(k_cache), a.vc = static_cast<const uint8_t *>(v_cache);
  a.table = page_table, a.kv_len = kv_len, a.cu_q = cu_q;
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.counters = static_cast<uint32_t *>(workspace);
  a.parts = static_cast<uint8_t *>(workspace) + kAttnCounters;
  a.table_width = d.table_width, a.table_s = d.table_s;
  // (without pages nothing is there, and nothing is read)
  a.most = d.pages ? (int32_t)std::min<int64_t>(d.table_width * d.page_size, INT32_MAX - 127) : 0;
  a.q_st = d.q_st, a.q_sh = d.q_sh, a.o_st = d.o_st, a.o_sh = d.o_sh;
  a.k_sp = d.k_sp, a.k_st = d.k_st, a.k_sh = d.k_sh;
  a.v_sp = d.v_sp, a.v_st = d.v_st, a.v_sh = d.v_sh;
  a.pages = (uint32_t)d.pages;
  a.g_mul = a.g_shift = 0;
  if (const int64_t G = d.Hq / d.Hkv; G > 1) { // ceil(2^(31 + s) / G), 2^s >= G
    const int sh = log2of(G);
    a.g_mul = (uint32_t)((((uint64_t)1 << (31 + sh)) + G - 1) / G), a.g_shift = sh - 1;
  }
  a.T = (int32_t)d.T, a.B = (int32_t)d.B, a.G = d.Hq / d.Hkv, a.Hq = d.Hq, a.Hkv = d.Hkv;
  a.head_dim = d.head_dim, a.page_shift = log2of(d.page_size);
  a.causal = d.causal, a.window = d.window;
  a.k_run = a.v_run = 0;
  a.qk_scale = d.sm_scale * 1.44269504f;
  g.ks = scalesOf(k_block_scale, s.k_sp, s.k_st, s.k_sh, s.k_sb);
  g.vs = scalesOf(v_block_scale, s.v_sp, s.v_st, s.v_sh, s.v_sb);
  g.packed = d.page_size >= 4 && aligned(k_block_scale, 4) && aligned(v_block_scale, 4) && s.k_st == 1 &&
             s.v_st == 1 && commonVec(4, {s.k_sp, s.k_sh, s.k_sb, s.v_sp, s.v_sh, s.v_sb}) == 4;
  const int D = attnDims(d.head_dim), di = D == 64 ? 0 : D == 96 ? 1 : D == 128 ? 2 : 3;
  const bool bf = d.dtype == TX_BF16, nv = s.mode == TX_SCALE_NV16;
  const Paged4AttnFn fn = plan->variant == 2 ? kPaged4Rows[di][bf][nv] : kPaged4Split[plan->variant][di][bf][nv];
  hipLaunchKernelGGL(fn, dim3(plan->grid_x), dim3(plan->block_threads), 0,
                     static_cast<hipStream_t>(stream), g);
  TX_HIP_CHECK(hipGetLastError());
  return TX_OK;
}
