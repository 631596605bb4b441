// Table of the attention over a 4-bit paged cache, many rows a sequence (paged_attn4.h).

#include "paged_attn4.h"

namespace txk {

typedef void (*Paged4AttnFn)(Paged4Args);
extern const Paged4AttnFn kPaged4Rows[4][2][2];

#define ROWS(D)                                                                                    \
  {{paged_attn4_rows_kernel<Paged4Rows<D, false, false>>,                                          \
    paged_attn4_rows_kernel<Paged4Rows<D, false, true>>},                                          \
   {paged_attn4_rows_kernel<Paged4Rows<D, true, false>>,                                           \
    paged_attn4_rows_kernel<Paged4Rows<D, true, true>>}}

// [64, 96, 128, 256 dims][bf16][e4m3 scales]
const Paged4AttnFn kPaged4Rows[4][2][2] = {ROWS(64), ROWS(96), ROWS(128), ROWS(256)};

} // namespace txk
