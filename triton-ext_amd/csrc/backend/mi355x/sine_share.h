// Which of a token's sines each thread of a workgroup forms (cache4_rows.h).  The same on the host, where a
// test goes through all forms.
#pragma once

#include <cstdint>

#include "tile_common.h"

namespace txk {

// Tokens have token_threads threads each, in workgroups of 256: whole tokens, or whole workgroups of
// one token, the last of which may have fewer (RotaryPlace).  A workgroup holds the sines of its
// tokens side by side; thread `thread`, the token's thread `in`, forms pairs first, first + step,
// .. of the workgroup's token `token`, so that the threads which the workgroup has form all of them.
struct SineShare {
  uint32_t token, first, step;
};
TX_HD SineShare sine_share(uint32_t thread, uint32_t token_threads, uint32_t in) {
  if (token_threads <= 256)
    return {thread / token_threads, in, token_threads};
  const uint32_t left = token_threads - (in - thread); // from this workgroup's first on
  return {0, thread, left < 256 ? left : 256};
}

} // namespace txk
