// How a product with a 4-bit weight is cut (linear4.hip): plain functions of its shape, also compiled for the host.
#pragma once
#include <stdint.h>

namespace kvh {

constexpr int kW4Rows = 16, kW4Block = 128;  // weight rows and k of a packed block

// Rows of x (in 16s) and weight tiles a wave holds, and the waves that share a tile's k.
struct Linear4Form {
  int mt, rt, wk;
};

inline Linear4Form linear4_form(int64_t tiles, int64_t blocks, int64_t m) {
  Linear4Form f;
  f.mt = m > 48 ? 4 : (int)((m + 15) / 16);
  f.rt = f.mt >= 3 || tiles >= 1024 ? 2 : 1;
  f.wk = blocks >= 16 && tiles / f.rt < 1024 ? 8 : 4;
  return f;
}

}  // namespace kvh
