// Which rows of a page each 1 KiB load of a block takes (paged_frag.h).  The same on the host, where a
// test goes through all forms.
#pragma once

#include <cstdint>
#include <type_traits>

#include "tile_common.h"

namespace txk {

// Rows of a load lie row & (run - 1) rows past the first of their run, with which the load's
// resource begins: `run` rows of a page, a power of two that divides it.
TX_HD uint32_t page_run_row(int row, int run) { return (uint32_t)(row & (run - 1)); }

// The loads `first` .. first + U - 1, R rows each, of a block.  resource(row): that of the run which
// begins with this row of the block.  load(u, rsrc, r0): load first + u, of the lanes whose row of
// it is r0 .. r0 + run - 1 (r0 < 0: of all lanes).
template <int U, int R, class Resource, class Load>
TX_HD void page_loads(int first, int run, Resource resource, Load load) {
  // N resources of U / N loads each
  auto fast = [&](auto count) __attribute__((always_inline)) {
    constexpr int N = decltype(count)::value;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const auto rsrc = resource(R * (first + U / N * i));
#pragma unroll
      for (int u = U / N * i; u < U / N * (i + 1); ++u)
        load(u, rsrc, -1);
    }
  };
  if (run >= U * R)
    fast(std::integral_constant<int, 1>());
  else if (U % 2 == 0 && 2 * run >= U * R)
    fast(std::integral_constant<int, U % 2 ? 1 : 2>());
  else if (U % 4 == 0 && 4 * run >= U * R)
    fast(std::integral_constant<int, U % 4 ? 1 : 4>());
  else { // runs of fewer rows; maybe fewer than a load has: the lanes of one at a time
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma nounroll
      for (int r0 = 0; r0 < R; r0 += run)
        load(u, resource((R * (first + u) + r0) & -run), run >= R ? -1 : r0);
  }
}

} // namespace txk
