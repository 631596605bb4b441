// Host harness for page_rows.h: goes through every form of a block's loads (rows of a load, loads of a
// wave, rows of a run) and prints "OK", or the first row that is not read from its own place.
#include <cstdio>
#include <vector>

#include "backend/mi355x/page_rows.h"

using namespace txk;

// A block of which each of `waves` waves takes U loads of R rows.  Row r lies in run r / run.
template <int U, int R> bool form(int waves, int run) {
  std::vector<int> times(waves * U * R, 0);
  bool ok = true;
  for (int w = 0; w < waves; ++w) {
    const int first = U * w;
    page_loads<U, R>(
        first, run,
        [&](int row) {
          if (row % run != 0) {
            printf("U=%d R=%d run=%d: a resource begins with row %d, inside a run\n", U, R, run, row);
            ok = false;
          }
          return row;
        },
        [&](int u, int begin, int r0) {
          for (int lr = 0; lr < R; ++lr) { // row of the load (all lanes of a row alike)
            if (r0 >= 0 && (lr < r0 || lr >= r0 + run))
              continue;
            const int row = R * (first + u) + lr, at = begin + (int)page_run_row(row, run);
            ++times[row];
            if (at != row && ok) {
              printf("U=%d R=%d run=%d: row %d is read from row %d's place\n", U, R, run, row, at);
              ok = false;
            }
          }
        });
  }
  for (size_t r = 0; r < times.size(); ++r)
    if (times[r] != 1 && ok) {
      printf("U=%d R=%d run=%d: row %zu is loaded %d times\n", U, R, run, r, times[r]);
      ok = false;
    }
  return ok;
}

// BN keys a block, shared by `waves` waves; LDS rows of ROW bytes; runs up to a wave's rows.
template <int ROW, int BN, int waves> bool forms() {
  constexpr int R = 1024 / ROW, U = BN / waves / R;
  static_assert(U > 0, "a load or more a wave");
  bool ok = true;
  for (int run = 1; run <= BN / waves; run *= 2)
    ok = form<U, R>(waves, run) && ok;
  return ok;
}

int main() {
  // 64 .. 256 dims of one or two bytes; a wave's own blocks of 32 keys, shared ones of 64
  bool ok = forms<64, 32, 1>();
  ok = forms<128, 32, 1>() && ok;
  ok = forms<256, 32, 1>() && ok;
  ok = forms<512, 32, 1>() && ok;
  ok = forms<64, 64, 4>() && ok;
  ok = forms<128, 64, 4>() && ok;
  ok = forms<256, 64, 4>() && ok;
  ok = forms<512, 64, 4>() && ok;
  if (!ok)
    return 1;
  printf("OK\n");
  return 0;
}
