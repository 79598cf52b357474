// Which tile a product of the block-scaled 8-bit GEMM takes, and in how many parts its sum over k is shared out. Plain C++ without
// HIP, so that the rule is checked over its whole range on the CPU.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace wanmi {

enum Fp8Tiles { kFp8Tiles64, kFp8Tiles128Deep, kFp8Tiles128, kFp8Tiles256 };

struct Fp8Plan {
  Fp8Tiles tiles;
  int splits;    // of the sum; the parts are added by a launch of their own
  int64_t cost;  // ns
};

constexpr int kFp8MaxSplits = 8;

// CUs that the choice counts with, whatever the device: the workspace of the parts is asked for before the call.
constexpr int64_t kFp8PlanCus = 256;

// Estimated time of M x N with KB blocks of 128 along the sum, from what was measured (weights from memory; us per stage of 128):
//   64 x 64, four stages in LDS, two workgroups a CU: 0.37, 0.55, 0.86, 1.06, 1.34 with 1 to 5 workgroups on the fullest CU
//   128 x 128, four stages, one workgroup a CU: 0.60 to 0.68 a round of 256
//   128 x 128, two stages, two workgroups a CU: 0.73 up to 256 tiles, 1.01 at 320, 1.36 at 432, 1.64 at 520
//   256 x 256, two stages, one workgroup a CU: 1.25 a round of 122 tiles, 1.87 a full one (the chip's power); 1.5 is counted for either
// So a CU gets through 35 to 65 KB/us of tiles, most with two workgroups or more (its loads could do 125: reading LDS and a barrier a stage are what takes the time), and
// what counts is how many bytes the fullest CU takes: small tiles and parts of the sum spread them, and read more. The parts are written and read once in fp32, at 6 TB/s, and a launch of 3.8 us adds them.
// (5120 x 5120: 20 rows 17.6 -> 12.1 us with three parts, 200 rows 24.1 -> 20.6, 333 rows, 4112 deep, 23.9 -> 22.7 with two; 512 rows 27.9
// and 38.6 with three: not taken. 13824 deep: 64 rows 41.2 -> 22.0, 200 rows 57.5 -> 34.1, 500 rows 67.1 -> 64.3.)
inline Fp8Plan fp8_plan(int64_t M, int64_t N, int64_t KB) {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t cus = kFp8PlanCus;
  const int64_t t64 = up(M, 64) * up(N, 64), t128 = up(M, 128) * up(N, 128), t256 = up(M, 256) * up(N, 256);
  Fp8Plan best{kFp8Tiles256, 1, 2500 + std::max<int64_t>(KB, 2) * 1500 * up(t256, cus)};
  auto take = [&](Fp8Tiles tiles, int splits, int64_t cost) {
    if (cost < best.cost) best = Fp8Plan{tiles, splits, cost};
  };
  take(kFp8Tiles128, 1, 2500 + std::max<int64_t>(KB, 2) * std::max<int64_t>(730, 780 * t128 / cus));
  for (int s = 1; s <= kFp8MaxSplits && s <= KB; ++s) {
    const int64_t stages = up(KB, s), join = s == 1 ? 0 : 3800 + s * M * N * 8 / 6000;
    take(kFp8Tiles64, s, 2500 + stages * (120 + 245 * up(t64 * s, cus)) + join);
    take(kFp8Tiles128Deep, s, 2500 + stages * 660 * up(t128 * s, cus) + join);
  }
  return best;
}

}  // namespace wanmi
