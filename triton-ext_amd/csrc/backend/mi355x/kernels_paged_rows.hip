// Table of the paged attention's kernels, many rows a sequence (paged_attn.h).

#include "paged_attn.h"

namespace txk {

typedef void (*PagedAttnFn)(PagedAttnArgs);
extern const PagedAttnFn kPagedAttnRows[4][2][2];
// [64, 96, 128, 256 dims][bf16][e4m3 cache]
const PagedAttnFn kPagedAttnRows[4][2][2] = {
    {{paged_attn_rows_kernel<PagedFrag<64, false, false, 64>>,
      paged_attn_rows_kernel<PagedFrag<64, false, true, 64>>},
     {paged_attn_rows_kernel<PagedFrag<64, true, false, 64>>,
      paged_attn_rows_kernel<PagedFrag<64, true, true, 64>>}},
    {{paged_attn_rows_kernel<PagedFrag<96, false, false, 64>>,
      paged_attn_rows_kernel<PagedFrag<96, false, true, 64>>},
     {paged_attn_rows_kernel<PagedFrag<96, true, false, 64>>,
      paged_attn_rows_kernel<PagedFrag<96, true, true, 64>>}},
    {{paged_attn_rows_kernel<PagedFrag<128, false, false, 64>>,
      paged_attn_rows_kernel<PagedFrag<128, false, true, 64>>},
     {paged_attn_rows_kernel<PagedFrag<128, true, false, 64>>,
      paged_attn_rows_kernel<PagedFrag<128, true, true, 64>>}},
    {{paged_attn_rows_kernel<PagedFrag<256, false, false, 64>>,
      paged_attn_rows_kernel<PagedFrag<256, false, true, 64>>},
     {paged_attn_rows_kernel<PagedFrag<256, true, false, 64>>,
      paged_attn_rows_kernel<PagedFrag<256, true, true, 64>>}}};

} // namespace txk
