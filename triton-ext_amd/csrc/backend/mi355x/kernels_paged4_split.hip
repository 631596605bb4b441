// Table of the attention over a 4-bit paged cache, up to 32 rows a sequence on average, heads of more than 64
// dims 64 (paged_attn4.h).

#include "paged_attn4.h"

namespace txk {

typedef void (*Paged4AttnFn)(Paged4Args);
extern const Paged4AttnFn kPaged4Split[2][4][2][2];

#define SPLIT(RT, D)                                                                               \
  {{paged_attn4_split_kernel<Paged4Split<D, false, false, RT>>,                                    \
    paged_attn4_split_kernel<Paged4Split<D, false, true, RT>>},                                    \
   {paged_attn4_split_kernel<Paged4Split<D, true, false, RT>>,                                     \
    paged_attn4_split_kernel<Paged4Split<D, true, true, RT>>}}

// [16, 32 rows][64, 96, 128, 256 dims][bf16][e4m3 scales]
const Paged4AttnFn kPaged4Split[2][4][2][2] = {
    {SPLIT(1, 64), SPLIT(1, 96), SPLIT(1, 128), SPLIT(1, 256)},
    {SPLIT(2, 64), SPLIT(2, 96), SPLIT(2, 128), SPLIT(2, 256)}};

} // namespace txk
