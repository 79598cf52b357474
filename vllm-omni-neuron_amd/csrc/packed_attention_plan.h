// Which tiles attention over packed rows takes. Plain C++ without HIP, so that the rule is checked over its whole range on the CPU.
#pragma once

#include <stdint.h>

namespace wanmi {

// True: tiles of 32 rows whose keys the four waves of a workgroup share out; false: tiles of 128 rows, 32 a wave, over the same keys.
// Shared keys pay where all tiles are on the chip at once (one to a CU with its 144 KB of LDS, two at head_dim 64) and there is more than a tile of 64 keys to
// share out: a row's chain of tiles is then a quarter as long. Past that 128 rows are as fast or faster, whether or not their waves all have rows: the
// tiles of 64 keys are loaded once for four waves. Each request is counted as one tile where they have 32 rows or fewer on average.
// us, shared / 128 rows, 40 heads x 128: 1 row of one request, 512 keys 10.2 / 13.5, 2000 keys 24.5 / 42.4, 64 keys 6.8 / 5.4; 4 requests of 32 rows,
// 512 keys 13.1 / 15.1; 8 of 1 row, 512 keys 24.7 / 21.4; 64 of 20 rows, 64 keys 57 / 29, 512 keys 160 / 135; 32 of 20 rows, 2000 keys 243 / 254; one of 3000 rows
// beside 127 single ones, 512 keys 397 / 268; 128 rows of one request, 512 keys 9.7 / 12.9; 200 rows 17.3 / 13.1. 64 heads x 64: 4 of 20 rows, 512 keys
// 9.0 / 11.5, 8 of 20 17.0 / 15.8, 16 of 20 28.0 / 33.7, 64 of 20, 64 keys 38 / 23. 12 heads x 64 with a bias: a prompt of 1024 tokens 12.9 / 20.8.
inline bool packed_keys_shared(int64_t T, int64_t Tk, int64_t requests, int64_t heads, int head_dim) {
  const int64_t tiles = (T <= 32 * requests ? requests : T / 32 + requests) * heads;
  return tiles <= (head_dim == 128 ? 256 : 512) && Tk > 64 * requests;
}

}  // namespace wanmi
