// Table of the paged attention's kernels, up to 16 rows a sequence (paged_attn.h).

#include "paged_attn.h"

namespace txk {

typedef void (*PagedAttnFn)(PagedAttnArgs);
extern const PagedAttnFn kPagedAttnSplit16[4][2][2];
// [64, 96, 128, 256 dims][bf16][e4m3 cache]
const PagedAttnFn kPagedAttnSplit16[4][2][2] = {
    {{paged_attn_split_kernel<PagedFrag16<64, false, false, 32>>,
      paged_attn_split_kernel<PagedFrag16<64, false, true, 32>>},
     {paged_attn_split_kernel<PagedFrag16<64, true, false, 32>>,
      paged_attn_split_kernel<PagedFrag16<64, true, true, 32>>}},
    {{paged_attn_split_kernel<PagedFrag16<96, false, false, 32>>,
      paged_attn_split_kernel<PagedFrag16<96, false, true, 32>>},
     {paged_attn_split_kernel<PagedFrag16<96, true, false, 32>>,
      paged_attn_split_kernel<PagedFrag16<96, true, true, 32>>}},
    {{paged_attn_split_kernel<PagedFrag16<128, false, false, 32>>,
      paged_attn_split_kernel<PagedFrag16<128, false, true, 32>>},
     {paged_attn_split_kernel<PagedFrag16<128, true, false, 32>>,
      paged_attn_split_kernel<PagedFrag16<128, true, true, 32>>}},
    {{paged_attn_split_kernel<PagedFrag16<256, false, false, 32>>,
      paged_attn_split_kernel<PagedFrag16<256, false, true, 32>>},
     {paged_attn_split_kernel<PagedFrag16<256, true, false, 32>>,
      paged_attn_split_kernel<PagedFrag16<256, true, true, 32>>}}};

} // namespace txk
