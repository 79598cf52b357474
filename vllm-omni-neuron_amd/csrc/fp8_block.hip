// Products with 8-bit weights that have one fp32 scale per block of 128 x 128, for gfx950.
//
//   y[m, n] = act( sum_b sa[m, b] sw[n / 128, b] sum_{k in block b} a[m, k] w[n, k] + bias[n] )
//
// a and w are e4m3 codes, b the blocks of 128 along k. The scales are any fp32 numbers, not powers of two, so the hardware's block
// scales cannot apply them: each block's inner product is one 16 x 16 x 128 MFMA from zero, and its result enters the fp32
// accumulator by a multiply-add with sa * sw (sw is the same for a wave's whole tile, and with the weight as the MFMA's first operand a lane's
// four results belong to one row m, so a block costs one factor per fragment). A multiply-add per result is half the time
// that its MFMA takes on the matrix pipe, and runs beside the other wave's MFMAs.
//
// Activations come as codes with scales, or as bf16 that is quantized on the way: amax of each 128 of a row (at least 2^-100) times
// fp32(1 / 448) is the scale, x / scale rounded to nearest the code. (bf16 values over their maximum fall onto the border between two codes often enough
// that the last bit of the scale decides many codes: the product with the rounded reciprocal is what torch computes on the GPU for `/ 448`.)
//
// Measured: 32760 x 15360 x 5120 from codes 2.15 ms, 2.4 PFLOP/s (a library's product of 8192^3 such codes with one scale reaches 3.0); the matrix
// pipe is busy 65% of the cycles, at 1.75 GHz, which the chip's power sets. 7799 x 5120 x 13824 from bf16 556 to 563 us, of which 53 quantize;
// 1560 x 13824 x 5120 136, of which 7; 333 x 5096 x 4112 26, in three launches of 4.8, 20.9 and 4.2.
#include "wanmi_common.h"
#include "fp8_plan.h"
#include "gemm_plan.h"

#include <algorithm>

namespace wanmi {

constexpr int kBlock = 128;

struct Fp8Args {
  const uint8_t* a;       // [M, lda] codes
  int64_t lda;
  const float* a_scales;  // block b of row m at m * as_row + b * as_blk
  int64_t as_row, as_blk;
  const uint16_t* x;      // bf16 [M, lda] in place of codes and scales (few rows)
  const uint8_t* w;       // [N, K]
  const float* w_scales;  // [ceil(N / 128), KB]
  const float* bias;      // [N] or null
  uint16_t* out;          // bf16 [M, ldo]
  int64_t ldo;
  int M, N, K, KB;
  int gelu;
  int tiles_m, tiles_n;
  int splits;             // of the sum over k, a workgroup each (kRing > 2)
  float* parts;           // [splits][M][N] where there are several
};

// As the MXFP8 GEMM's: gelu_tanh(x) = x / (1 + 2^(x (k0 + k1 x^2))).
__device__ __forceinline__ float gelu_tanh_f32(float x) {
  const float e = __builtin_amdgcn_exp2f(x * (-2.302208198144325f + -0.1029432395800235f * (x * x)));
  return x * __builtin_amdgcn_rcpf(1.0f + e);
}

// ------------------------------------------------------------------------------------------------
// Quantization
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t max_magnitude(uint32_t best, uint32_t pair) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, best), __builtin_bit_cast(u16x2_t, pair & 0x7FFF7FFFu)));
}
// The scale of a block from its largest magnitude (bf16 bits; those of infinities and NaN are the largest, and then every code of the block is NaN).
__device__ __forceinline__ float block_scale(uint32_t best) {
  const uint32_t top = max(best >> 16, best & 0xFFFFu);
  const float amax = bf16_to_f32((uint16_t)top);
  return (amax < 0x1p-100f ? 0x1p-100f : amax) * (1.0f / 448.0f);
}
// x / scale rounded as the division rounds it: with y the rounded reciprocal, q + (x - q scale) y rounds correctly for q = x y (Markstein);
// nothing here underflows that could reach a code (scales are 2^-109 or more).
__device__ __forceinline__ float quotient(float x, float scale, float y) {
  const float q = x * y;
  return fmaf(fmaf(-q, scale, x), y, q);
}
__device__ __forceinline__ uint32_t four_codes(uint32_t p01, uint32_t p23, float scale, float y) {
  return cvt_e4m3x4(quotient(bf16_lo(p01), scale, y), quotient(bf16_hi(p01), scale, y), quotient(bf16_lo(p23), scale, y),
                    quotient(bf16_hi(p23), scale, y));
}

// The largest magnitude over 16 lanes: quad permutes, then the half-row and row mirrors, which pair equal quads.
__device__ __forceinline__ uint32_t max_of_16_lanes(uint32_t best) {
  best = max_magnitude(best, (uint32_t)dpp_i32<0xB1>((int)best));
  best = max_magnitude(best, (uint32_t)dpp_i32<0x4E>((int)best));
  best = max_magnitude(best, (uint32_t)dpp_i32<0x141>((int)best));
  return max_magnitude(best, (uint32_t)dpp_i32<0x140>((int)best));
}

// A workgroup takes four blocks of 32 rows, a wave four of the rows with all loads under way together, 16 lanes x 8 values to a block. The
// scales leave by way of LDS, so that block by block the 32 rows' are one whole line (by itself each is 4 bytes of a line that
// eight XCDs write to). K is a multiple of 16: a lane's 8 values are all inside or all behind. Memory bounds it: 7799 x 13824, 327 MB, take 53 us,
// 6.2 TB/s (a copy of that size 5.4); one row's load at a time and scales straight to memory took 62.
constexpr int kQuantRows = 32, kQuantBlocks = 4;
__global__ __launch_bounds__(512) void fp8_block_quantize_kernel(const uint16_t* __restrict__ x, int64_t ldx, int M, int K, int KB,
                                                                uint8_t* __restrict__ codes, float* __restrict__ scales,
                                                                int64_t s_row, int64_t s_blk) {
  constexpr int kOwn = kQuantRows / 8;  // rows of a wave
  __shared__ float turn[kQuantBlocks][kQuantRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int units = (KB + kQuantBlocks - 1) / kQuantBlocks;
  const int group = (int)blockIdx.x / units, b0 = ((int)blockIdx.x - group * units) * kQuantBlocks;
  const int64_t m0 = (int64_t)group * kQuantRows;
  const int row = wave * kOwn, k = (b0 + (lane >> 4)) * kBlock + 8 * (lane & 15);
  u32x4 v[kOwn];
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    v[u] = u32x4{0u, 0u, 0u, 0u};
    if (k < K && m0 + row + u < M) v[u] = *reinterpret_cast<const u32x4*>(x + (m0 + row + u) * ldx + k);
  }
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) best = max_magnitude(best, v[u][i]);
    const float scale = block_scale(max_of_16_lanes(best)), y = 1.0f / scale;
    if (k < K && m0 + row + u < M)
      *reinterpret_cast<uint2*>(codes + (m0 + row + u) * K + k) = make_uint2(four_codes(v[u][0], v[u][1], scale, y), four_codes(v[u][2], v[u][3], scale, y));
    if ((lane & 15) == 0) turn[lane >> 4][row + u] = scale;
  }
  __syncthreads();
  const int b = threadIdx.x / kQuantRows, r = threadIdx.x % kQuantRows;
  if (b < kQuantBlocks && b0 + b < KB && m0 + r < M) scales[(m0 + r) * s_row + (b0 + b) * s_blk] = turn[b][r];
}

// scales [M, KB] of any strides -> [KB, M]
__global__ __launch_bounds__(256) void fp8_scales_kernel(const float* __restrict__ in, int64_t s_row, int64_t s_blk, int M, int KB, float* __restrict__ out) {
  const int m = blockIdx.x * 64 + (threadIdx.x & 63);
  if (m >= M) return;
  for (int b = threadIdx.x >> 6; b < KB; b += 4) out[(int64_t)b * M + m] = in[m * s_row + b * s_blk];
}

// ------------------------------------------------------------------------------------------------
// Many rows: tiles of kTn features x kTm rows, both operands through LDS in stages of 128 along k. The matrix pipe and the chip's power bound the
// 256 x 256 tiles: 32760 x 15360 x 5120 took 2912 us with the multiply-adds where the compiler put them, 2380 in the order below, 2322 without
// bank conflicts, 2150 with workgroups that stay and addresses in scalar registers (16 to 23 of them wait in lanes of a vector register between tiles; the
// stages' loop reads none of them back, in the 64 x 64 tiles one). A full round of 256 tiles costs 1.87 us a stage, one
// of 122 tiles 1.25: cutting the last round's tiles in parts of their sums or in halves gained nothing. The smaller tiles are
// bound by LDS (128 x 128: 96 KB read and 32 written a stage, 1024 of 1340 cycles) and the stage's barrier.
// ------------------------------------------------------------------------------------------------
// 16-byte chunk c of row r lies in slot c ^ f(r) of its 128 bytes. One cycle of a 16-byte read serves lanes 0-3, 12-15 and 20-27 (or the others
// of 32): all sixteen rows of a fragment, chunk q of rows 0-3 and 12-15 and chunk q ^ 1 of rows 4-11. Two rows share the 64 banks, so
// the eight even and the eight odd rows each need eight slots: f(r) ^ (r in 4..11) has to be one to one on them.
__device__ __forceinline__ int fp8_slot(int row) { return (row & 7) ^ ((row >> 2) & 1); }

// What one tile's loads need: the wave's operand (the first half of the waves loads the weight, the second the rows), the scales.
struct Fp8Tile {
  uint64_t src, scales, wscales;
  uint32_t src_bytes, scales_bytes, wscales_bytes;  // 0: no tile, nothing moves
  int m0, n0;
};

// 64 bits of address, 32 of extent, all the same in every lane
__device__ __forceinline__ u32x4 uniform_rsrc(uint64_t base, uint32_t bytes) {
  return u32x4{(uint32_t)base, (uint32_t)(base >> 32) & 0xFFFFu, bytes, 0x00020000u};
}
// (the same in every lane, but where the compiler does not prove it it keeps it in vector registers)
__device__ __forceinline__ u32x4 first_lane_rsrc(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) & 0xFFFFu,
               (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}
__device__ __forceinline__ float uniform_load(uint64_t base, uint32_t bytes, int off) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
  return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}

template <int kTn, int kTm, int kWn, int kWm, int kRing>  // the tile, how many waves along each side, stages in LDS
__global__ __launch_bounds__(64 * kWn * kWm, 2) void fp8_block_gemm_kernel(Fp8Args g) {
  static_assert(kTn == kTm, "half of the waves loads either operand");
  constexpr int kWaves = kWn * kWm;
  constexpr int kFn = kTn / kWn / 16, kFm = kTm / kWm / 16;  // fragments of a wave
  constexpr int kStage = (kTn + kTm) * kBlock;
  constexpr int kLoads = (kTn + kTm) / 8 / kWaves;           // per wave and stage
  constexpr int kLoadsLast = kFn == 8 ? 2 : kFn == 4 ? 4 : kLoads;  // of them in a stage's last row, and as many in each of the next rows
  static_assert(kFn % 2 == 0 && kLoads % kLoadsLast == 0 && kLoads / kLoadsLast < kFn, "fragments alternate; loads end before the wait for them");
  constexpr int kRow = 32 * kFn;         // bytes of a wave's output row
  constexpr int kStaging = 16 * kRow;    // sixteen rows
  // The scales of a stage: into registers one stage ahead, or with more stages in LDS through it as well (the compiler waits for loads into
  // registers as if there were no others under way, for all of them).
  constexpr bool kLdsScales = kRing > 2;
  constexpr int kScales = kLdsScales ? 4 * kTm + 512 : 0;  // bytes: of the rows, of the weight (256, one value counts), unused
  constexpr int kStageLoads = kLoads + (kLdsScales ? 1 : 0);
  static_assert(!kLdsScales || (kTn <= kBlock && kTm / 64 < kWaves), "one weight scale a tile; a wave each for the loads of the scales");
  static_assert(kStaging >= 1024, "a load of the bias fits");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kRing * (kStage + kScales)];
  __shared__ __attribute__((aligned(1024))) uint8_t staging[kWaves * kStaging];
  constexpr int kScalesAt = kRing * kStage;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, q = lane >> 4;
  const int mw = (wave % kWm) * 16 * kFm, nw = (wave / kWm) * 16 * kFn;  // the wave's first row and feature
  const bool weight = wave < kWaves / 2;
  const uint32_t ld = weight ? (uint32_t)g.K : (uint32_t)g.lda;
  const uint32_t row0 = (uint32_t)(wave % (kWaves / 2)) * (8 * kLoads);  // of the rows it loads
  const int total = g.tiles_m * g.tiles_n;
  // the stages of the workgroup's part of the sum: [first, first + stages)
  const int split = kRing > 2 ? (int)(blockIdx.x / (unsigned)total) : 0;
  const int first = kRing > 2 ? (int)((int64_t)g.KB * split / g.splits) : 0;
  const int stages = kRing > 2 ? (int)((int64_t)g.KB * (split + 1) / g.splits) - first : max(g.KB, 2);  // (the second of one block's two reads zeros)

  auto tile_of = [&](int v) {
    Fp8Tile t;
    const TileAt at = tile_at(min(v, total - 1), g.tiles_m, g.tiles_n, kGroupM * TM / kTm);
    t.m0 = at.tm * kTm;
    t.n0 = at.tn * kTn;
    const int mv = min(kTm, g.M - t.m0), nv = min(kTn, g.N - t.n0);
    const bool some = v < total;
    t.src = weight ? reinterpret_cast<uint64_t>(g.w) + (uint64_t)t.n0 * (uint64_t)g.K : reinterpret_cast<uint64_t>(g.a) + (uint64_t)t.m0 * (uint64_t)g.lda;
    t.src_bytes = some ? (uint32_t)((weight ? nv : mv) - 1) * ld + (uint32_t)g.K : 0u;
    t.scales = reinterpret_cast<uint64_t>(g.a_scales + t.m0);  // (as_row is 1)
    t.scales_bytes = some ? (uint32_t)mv * 4 : 0u;
    t.wscales = reinterpret_cast<uint64_t>(g.w_scales + (int64_t)(min(t.n0 + nw, g.N - 1) / kBlock) * g.KB);
    t.wscales_bytes = some ? (uint32_t)g.KB * 4 : 0u;
    return t;
  };

  // rows 8 i + (lane >> 3) from row0 on; slot lane & 7 takes the chunk whose slot that is; chunks behind K read as zeros
  const uint32_t lchunk = (uint32_t)(((lane & 7) ^ fp8_slot(lane >> 3)) << 4);
  const uint32_t lvoff = (uint32_t)(lane >> 3) * ld + lchunk;
  uint64_t load_base;  // of the stage that is being loaded
  uint32_t load_bytes, load_voff, load_to;
  auto begin_stage = [&](uint64_t src, uint32_t bytes, int kt, int buffer) {
    const uint32_t off = row0 * ld + (uint32_t)kt * kBlock;
    load_base = src + off;
    load_bytes = max((int)(bytes - off), 0);
    load_voff = lchunk + (uint32_t)kt * kBlock < (uint32_t)g.K ? lvoff : 0xFFFFFFF0u;
    load_to = lds_addr(lds) + (uint32_t)buffer * kStage + (uint32_t)(wave * kLoads) * 1024;
  };
  auto load = [&](int i) {
    const uint32_t off = (uint32_t)(8 * i) * ld;
    lds_dma_b128_hot(uniform_rsrc(load_base + off, (uint32_t)max((int)(load_bytes - off), 0)), load_voff, load_to + i * 1024);
  };
  float sa[kFm], sw;
  auto load_scales = [&](uint64_t rows, uint32_t rows_bytes, uint64_t ws, uint32_t ws_bytes, int kt) {
    kt = min(kt, g.KB - 1);
    const uint64_t base = rows + (uint64_t)kt * ((uint64_t)g.as_blk * 4);
#pragma unroll
    for (int j = 0; j < kFm; ++j) sa[j] = uniform_load(base, rows_bytes, (mw + c) * 4 + 64 * j);
    sw = uniform_load(ws + (uint64_t)kt * 4, ws_bytes ? 4u : 0u, 0);
  };
  // the wave's part of a stage's scales: 64 rows', the weight's one, or nothing
  auto dma_scales = [&](uint64_t rows, uint32_t rows_bytes, uint64_t ws, uint32_t ws_bytes, int kt, int buffer) {
    if constexpr (kLdsScales) {
      const bool row = wave < kTm / 64, one = wave == kTm / 64;
      kt = min(kt, g.KB - 1);
      const uint64_t base = row ? rows + (uint64_t)kt * ((uint64_t)g.as_blk * 4) + 256 * wave : ws + (uint64_t)kt * 4;
      const uint32_t bytes = row ? (uint32_t)max((int)rows_bytes - 256 * wave, 0) : one && ws_bytes ? 4u : 0u;
      lds_dma_b32(uniform_rsrc(base, bytes), (uint32_t)lane * 4, lds_addr(lds) + kScalesAt + buffer * kScales + (row ? 256 * wave : one ? 4 * kTm : 4 * kTm + 256));
    }
  };
  auto read_scales = [&](int buffer) {
    const float* p = reinterpret_cast<const float*>(lds + kScalesAt + buffer * kScales);
#pragma unroll
    for (int j = 0; j < kFm; ++j) sa[j] = p[mw + c + 16 * j];
    sw = p[kTm];
  };
  // lane's bytes of a row: chunks q and 4 + q (in both operands, so the order of k is of no account)
  const int o0 = c * kBlock + ((q ^ fp8_slot(c)) << 4), o1 = c * kBlock + (((4 + q) ^ fp8_slot(c)) << 4);
  auto fragment = [&](int buffer, int row) {
    const uint8_t* p = lds + buffer * kStage + row * kBlock;
    const u32x4 x = *reinterpret_cast<const u32x4*>(p + o0), y = *reinterpret_cast<const u32x4*>(p + o1);
    return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
  };

  // A stage is kFn rows of kFm MFMAs (one weight fragment each). Beside an MFMA run the multiply-adds of the same column's MFMA one row
  // before, the reads of the next row's weight fragment and the loads of the stages ahead, in this order (the scheduling barriers keep it: left
  // to itself the compiler put every multiply-add right behind its MFMA and waited). Before the last row every wave has read all of its stage
  // and the next one is in LDS: the one barrier of a stage. The last row then reads the next stage's first fragments, and the stage
  // after next is loaded into the buffer from there on. A tile's last stages load the first ones of the workgroup's next tile, so that only the
  // epilogue's own work is between two tiles.
  int v = (int)blockIdx.x - split * total;
  Fp8Tile t = tile_of(v), tn = tile_of(v + gridDim.x);
  int buf = 0;  // buffer of the stage
  if constexpr (!kLdsScales) load_scales(t.scales, t.scales_bytes, t.wscales, t.wscales_bytes, 0);
#pragma unroll
  for (int st = 0; st < kRing; ++st) {  // (of the last one of them only what a last row loads)
    begin_stage(t.src, st < stages ? t.src_bytes : 0u, first + st, st);
    dma_scales(t.scales, t.scales_bytes, t.wscales, t.wscales_bytes, first + st, st);
#pragma unroll
    for (int i = 0; i < (st < kRing - 1 ? kLoads : kLoadsLast); ++i) load(i);
  }
  constexpr int kFirstWait = (kRing - 2) * kStageLoads + kLoadsLast + (kLdsScales ? 1 : 0);  // loads behind the first stage's
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(kFirstWait));
  __syncthreads();
  f32x4 acc[kFn][kFm], p[kFm];
  float s[kFm];
  i32x8 fa[kFm], fw[2];
#pragma unroll
  for (int j = 0; j < kFm; ++j) fa[j] = fragment(0, kTn + mw + 16 * j);
  fw[0] = fragment(0, nw);
  if constexpr (kLdsScales) read_scales(0);

  for (;;) {
#pragma unroll
    for (int j = 0; j < kFm; ++j) {
      p[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      s[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < kFn; ++i) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int kt = 0; kt < stages; ++kt) {
#pragma unroll
      for (int i = 0; i < kFn; ++i) {
        const bool last = i == kFn - 1;
        if (last) {
          __builtin_amdgcn_s_waitcnt(waitcnt_lgkm(0));
          __builtin_amdgcn_s_waitcnt(waitcnt_vm((kRing - 2) * kStageLoads));
          __syncthreads();
          if constexpr (!kLdsScales) {
            // the scales of the next stage are here: the compiler's own wait for them belongs here too, not behind the loads below
#pragma unroll
            for (int j = 0; j < kFm; ++j) asm volatile("" : "+v"(sa[j]));
            asm volatile("" : "+v"(sw));
          }
          const bool here = kt + kRing < stages;  // (selected, not branched)
          const int ahead = here ? kt + kRing : kt + kRing - stages;
          if constexpr (kRing == 2) {
            begin_stage(here ? t.src : tn.src, here ? t.src_bytes : tn.src_bytes, ahead, buf);
          } else {  // (no next tile)
            begin_stage(t.src, here ? t.src_bytes : 0u, first + ahead, buf);
            dma_scales(t.scales, t.scales_bytes, t.wscales, t.wscales_bytes, first + ahead, buf);
          }
        }
        const int next = buf + 1 == kRing ? 0 : buf + 1;
        fw[(i + 1) & 1] = last ? fragment(next, nw) : fragment(buf, nw + 16 * (i + 1));
        if (kLdsScales && last) read_scales(next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kFm; ++j) {
          const int prev = i == 0 ? kFn - 1 : i - 1;
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[prev][j][r] = fmaf(p[j][r], s[j], acc[prev][j][r]);
          if (i == 0) s[j] = sa[j] * sw;  // of this stage, from here on
          const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
          p[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[i & 1], fa[j], zero, 0, 0, 0, 0, 0, 0);
          if (last) fa[j] = fragment(next, kTn + mw + 16 * j);
#pragma unroll
          for (int l = j * kLoadsLast / kFm; l < (j + 1) * kLoadsLast / kFm; ++l) {
            const int at = last ? l : kLoadsLast * (i + 1) + l;
            if (at < kLoads) load(at);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (i == 0) {
          [[maybe_unused]] const bool here = kt + 1 < stages;
          if constexpr (!kLdsScales) load_scales(here ? t.scales : tn.scales, here ? t.scales_bytes : tn.scales_bytes, here ? t.wscales : tn.wscales,
                      here ? t.wscales_bytes : tn.wscales_bytes, here ? kt + 1 : 0);
          // the bias of the wave's features, where its first output rows will be staged
          if (kt == 0)
            lds_dma_b128(first_lane_rsrc(g.bias + t.n0 + nw, g.bias ? (uint32_t)min(max(g.N - t.n0 - nw, 0), 16 * kFn) * 4 : 0u),
                         (uint32_t)lane * 16, lds_addr(staging) + wave * kStaging);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      buf = buf + 1 == kRing ? 0 : buf + 1;
    }
#pragma unroll
    for (int j = 0; j < kFm; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[kFn - 1][j][r] = fmaf(p[j][r], s[j], acc[kFn - 1][j][r]);

    if constexpr (kRing > 2) wait_vm<0>();  // the bias: the waits of a short sum may not have reached it
    // ---- epilogue: lane holds features nw + 16 i + 4 q .. + 3 of row mw + 16 j + c. Sixteen rows at a time are staged in the wave's LDS
    // and stored whole, past L2: they are written once and read by the next kernel ----
    if (kRing > 2 && g.splits > 1) {
      // a part of the sum, in fp32: fp8_join_kernel adds them
      float* po = g.parts + ((int64_t)split * g.M + t.m0 + mw + c) * g.N + t.n0 + nw + 4 * q;
#pragma unroll
      for (int j = 0; j < kFm; ++j)
#pragma unroll
        for (int i = 0; i < kFn; ++i)
          if (t.m0 + mw + 16 * j + c < g.M && t.n0 + nw + 16 * i + 4 * q < g.N)
            store_b128_guarded(__builtin_bit_cast(u32x4, acc[i][j]), po + (int64_t)16 * j * g.N + 16 * i);
      return;
    }
    constexpr int kCh = kRow / 16, kPer = 64 / kCh;  // chunks of a row, rows of a store
    uint8_t* stage = staging + wave * kStaging;
    const int el = fresh_lane_id(), ec = el & 15, eq = el >> 4;  // (nothing of the epilogue is held through the loop)
#pragma unroll
    for (int i = 0; i < kFn; ++i) {
      const f32x4 b = *reinterpret_cast<const f32x4*>(stage + 64 * i + 16 * eq);
#pragma unroll
      for (int j = 0; j < kFm; ++j) acc[i][j] += b;
    }
    const int rows = min(max(g.M - t.m0 - mw, 0), 16 * kFm);
    const uint64_t po = reinterpret_cast<uint64_t>(g.out + (int64_t)(t.m0 + mw) * g.ldo + t.n0 + nw);
    // (the same in every lane, which the compiler does not prove: without this each store became a loop over the lanes' values)
    const uint32_t plo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)po), phi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(po >> 32));
    const uint64_t pu = ((uint64_t)phi << 32) | plo;
    const auto ro = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(pu), (short)0, (int)__builtin_amdgcn_readfirstlane((uint32_t)rows * (uint32_t)g.ldo * 2), 0x00020000);
    const int ch = el % kCh;
    const bool in = t.n0 + nw + 8 * ch < g.N;
#pragma unroll
    for (int j = 0; j < kFm; ++j) {
#pragma unroll
      for (int i = 0; i < kFn; ++i) {
        float y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[r] = acc[i][j][r];
          if (g.gelu) y[r] = gelu_tanh_f32(y[r]);
        }
        *reinterpret_cast<uint2*>(stage + ec * kRow + (((2 * i + (eq >> 1)) ^ (ec & (kCh - 1))) << 4) + 8 * (eq & 1)) =
            make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
      }
#pragma unroll
      for (int it = 0; it < 16 / kPer; ++it) {
        const int r = it * kPer + el / kCh;
        const u32x4 d = *reinterpret_cast<const u32x4*>(stage + r * kRow + ((ch ^ (r & (kCh - 1))) << 4));
        const uint32_t off = (uint32_t)(16 * j + r) * (uint32_t)g.ldo * 2 + (uint32_t)ch * 16;  // (rows past M are dropped)
        __builtin_amdgcn_raw_buffer_store_b128(d, ro, (int)(in ? off : 0xFFFFFFF0u), 0, 2);
      }
    }
    v += gridDim.x;
    if (v >= total) break;
    t = tn;
    tn = tile_of(v + gridDim.x);
  }
  __builtin_amdgcn_s_waitcnt(0);  // no load may still be under way to LDS when the workgroup ends
}

// out = act(sum of the parts, in their order, + bias): eight columns a thread. Two parts of 333 x 5096 take 4.2 us, a launch's worth.
__global__ __launch_bounds__(256) void fp8_join_kernel(const float* __restrict__ parts, int splits, int M, int N, const float* __restrict__ bias, int gelu,
                                                      uint16_t* __restrict__ out, int64_t ldo) {
  const int per_row = N / 8;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = id / per_row;
  if (m >= M) return;
  const int n = (int)(id - m * per_row) * 8;
  f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f}, b = a;
  const float* p = parts + m * N + n;
  for (int s = 0; s < splits; ++s, p += (int64_t)M * N) {
    a += *reinterpret_cast<const f32x4*>(p);
    b += *reinterpret_cast<const f32x4*>(p + 4);
  }
  if (bias) {
    a += *reinterpret_cast<const f32x4*>(bias + n);
    b += *reinterpret_cast<const f32x4*>(bias + n + 4);
  }
  if (gelu) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      a[r] = gelu_tanh_f32(a[r]);
      b[r] = gelu_tanh_f32(b[r]);
    }
  }
  store_b128_guarded(u32x4{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])}, out + m * ldo + n);
}

// ------------------------------------------------------------------------------------------------
// Few rows: a workgroup of eight waves takes 16 features and all rows, the waves share out the blocks of k. What counts is to read the weight
// once, at the memory's rate: all loads of a wave are under way together, whole 128-byte lines of eight rows to an instruction (in the
// MFMA's own layout, half lines of sixteen rows, a launch that only read took 5.7 us in place of 2.7 on 26 MB in the caches, 7.0 and 5.9 from
// memory), and each block then goes through 2 KB of the wave's LDS into that layout.
// Rows in bf16 are quantized by the wave that needs them, 16 lanes to a block of a row; more than four of them in a launch of their own before
// (16 rows here would cost every workgroup as much again as its loads). One row of bf16 by 5120 x 5120, 26 MB: 7.6 us with the weight in the
// caches, 11.1 from memory.
// ------------------------------------------------------------------------------------------------
constexpr int kFewWaves = 8;
constexpr int kFewAhead = 5;      // blocks under way in a wave
constexpr int kFewRows = 16;      // at most
constexpr int kFewQuantize = 4;   // of them in bf16

__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off, bool in) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(in ? off : 0xFFFFFFF0u), 0, 0));
}

template <bool kQuantize>
__global__ __launch_bounds__(64 * kFewWaves, 2) void fp8_block_few_kernel(Fp8Args g) {
  constexpr int kPasses = kFewAhead * kFewQuantize / 4;  // four blocks of a row at a time
  __shared__ f32x4 red[kFewWaves][64];
  __shared__ __attribute__((aligned(16))) uint8_t turn[kFewWaves][16 * kBlock];
  __shared__ __attribute__((aligned(16))) uint8_t codes[kQuantize ? kFewWaves : 1][kQuantize ? 4 * kPasses * kBlock : 16];
  __shared__ float scales[kQuantize ? kFewWaves : 1][kQuantize ? 4 * kPasses : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, q = lane >> 4, r8 = lane >> 3, c8 = lane & 7;
  const int n0 = blockIdx.x * 16;
  // (rows behind N and chunks behind K read as zeros)
  const auto rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(g.w) + (int64_t)n0 * g.K, (short)0, min(16, g.N - n0) * g.K, 0x00020000);
  const void* rows = kQuantize ? (const void*)g.x : (const void*)g.a;
  const int row_bytes = (int)g.lda * (kQuantize ? 2 : 1), k_bytes = g.K * (kQuantize ? 2 : 1);
  const auto rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(rows), (short)0, (g.M - 1) * row_bytes + k_bytes, 0x00020000);
  const float* psw = g.w_scales + (int64_t)(n0 / kBlock) * g.KB;
  const int row = min(c, g.M - 1);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};

  for (int b0 = wave; b0 < g.KB; b0 += kFewWaves * kFewAhead) {
    u32x4 w[kFewAhead][2], x[kQuantize ? kPasses : kFewAhead][2];
    float sw[kFewAhead], sx[kFewAhead];
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      const int k = (b0 + kFewWaves * u) * kBlock + 16 * c8;
      w[u][0] = load16(rw, (uint32_t)(r8 * g.K + k), k < g.K);
      w[u][1] = load16(rw, (uint32_t)((8 + r8) * g.K + k), k < g.K);
    }
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      const int b = min(b0 + kFewWaves * u, g.KB - 1);
      sw[u] = psw[b];
      if constexpr (!kQuantize) {
        const int k = (b0 + kFewWaves * u) * kBlock + 16 * q;
        x[u][0] = load16(rx, (uint32_t)(row * row_bytes + k), k < g.K);
        x[u][1] = load16(rx, (uint32_t)(row * row_bytes + k + 64), k + 64 < g.K);
        sx[u] = g.a_scales[row * g.as_row + b * g.as_blk];
      }
    }
    if constexpr (kQuantize) {
      // block i of the batch's M * kFewAhead: block i % kFewAhead of row i / kFewAhead; 8 values a lane
      const int blocks = g.M * kFewAhead;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const int i = 4 * p + q, m = i / kFewAhead, k = (b0 + kFewWaves * (i - m * kFewAhead)) * kBlock + 8 * c;
        if (4 * p < blocks) x[p][0] = load16(rx, (uint32_t)(m * row_bytes + 2 * k), i < blocks && k < g.K);
      }
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        if (4 * p >= blocks) break;
        uint32_t best = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) best = max_magnitude(best, x[p][0][e]);
        const float s = block_scale(max_of_16_lanes(best)), y = 1.0f / s;
        const int i = 4 * p + q;
        *reinterpret_cast<uint2*>(&codes[wave][i * kBlock + 8 * c]) = make_uint2(four_codes(x[p][0][0], x[p][0][1], s, y), four_codes(x[p][0][2], x[p][0][3], s, y));
        if (c == 0) scales[wave][i] = s;
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // (the compiler sank the loads to their uses)
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      // into the MFMA's layout: row c's chunks q and 4 + q (a wave's LDS operations complete in order)
      uint8_t* t = turn[wave];
      *reinterpret_cast<u32x4*>(t + r8 * kBlock + ((c8 ^ fp8_slot(r8)) << 4)) = w[u][0];
      *reinterpret_cast<u32x4*>(t + (8 + r8) * kBlock + ((c8 ^ fp8_slot(r8)) << 4)) = w[u][1];
      const u32x4 w0 = *reinterpret_cast<const u32x4*>(t + c * kBlock + ((q ^ fp8_slot(c)) << 4));
      const u32x4 w1 = *reinterpret_cast<const u32x4*>(t + c * kBlock + (((4 + q) ^ fp8_slot(c)) << 4));
      const i32x8 fw = {(int)w0[0], (int)w0[1], (int)w0[2], (int)w0[3], (int)w1[0], (int)w1[1], (int)w1[2], (int)w1[3]};
      u32x4 x0, x1;
      float s;
      if constexpr (kQuantize) {
        const int i = row * kFewAhead + u;
        x0 = *reinterpret_cast<const u32x4*>(&codes[wave][i * kBlock + 16 * q]);
        x1 = *reinterpret_cast<const u32x4*>(&codes[wave][i * kBlock + 64 + 16 * q]);
        s = scales[wave][i];
      } else {
        x0 = x[u][0], x1 = x[u][1];
        s = sx[u];
      }
      const i32x8 fa = {(int)x0[0], (int)x0[1], (int)x0[2], (int)x0[3], (int)x1[0], (int)x1[1], (int)x1[2], (int)x1[3]};
      s = b0 + kFewWaves * u < g.KB ? s * sw[u] : 0.0f;  // (blocks behind the last have codes of zero)
      const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
      const f32x4 p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw, fa, zero, 0, 0, 0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = fmaf(p[r], s, acc[r]);
    }
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave > 0) return;  // the parts in the waves' order
  f32x4 y = red[0][lane];
#pragma unroll
  for (int w = 1; w < kFewWaves; ++w) y += red[w][lane];
  const int n = n0 + 4 * q;
  if (c >= g.M || n >= g.N) return;
  if (g.bias) y += *reinterpret_cast<const f32x4*>(g.bias + n);
  if (g.gelu) {
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = gelu_tanh_f32(y[r]);
  }
  *reinterpret_cast<uint2*>(g.out + (int64_t)c * g.ldo + n) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
}

static void launch_quantize(const uint16_t* x, int64_t ldx, int M, int K, uint8_t* codes, float* scales, int64_t s_row, int64_t s_blk, hipStream_t st) {
  const int KB = (K + kBlock - 1) / kBlock;
  const int64_t wgs = ((int64_t)M + kQuantRows - 1) / kQuantRows * ((KB + kQuantBlocks - 1) / kQuantBlocks);
  hipLaunchKernelGGL(fp8_block_quantize_kernel, dim3((unsigned)wgs), dim3(512), 0, st, x, ldx, M, K, KB, codes, scales, s_row, s_blk);
}

template <int kTn, int kTm, int kWn, int kWm, int kRing>
static void launch_tiles(Fp8Args g, int64_t wgs, hipStream_t st) {  // wgs: that walk the tiles; with more than two stages each tile (and part) has its own
  g.tiles_m = (g.M + kTm - 1) / kTm;
  g.tiles_n = (g.N + kTn - 1) / kTn;
  const int64_t total = (int64_t)g.tiles_m * g.tiles_n;
  hipLaunchKernelGGL((fp8_block_gemm_kernel<kTn, kTm, kWn, kWm, kRing>), dim3((unsigned)(kRing > 2 ? total * g.splits : std::min(total, wgs))),
                     dim3(64 * kWn * kWm), 0, st, g);
  if (kRing > 2 && g.splits > 1)
    hipLaunchKernelGGL(fp8_join_kernel, dim3((unsigned)(((int64_t)g.M * (g.N / 8) + 255) / 256)), dim3(256), 0, st, g.parts, g.splits, g.M, g.N, g.bias, g.gelu,
                       g.out, g.ldo);
}

static int64_t blocks_of(int64_t K) { return (K + kBlock - 1) / kBlock; }

static int check_sizes(int64_t M, int64_t K, const char* what) {
  WANMI_REQUIRE(M >= 0 && M < (1LL << 27), WANMI_ERR_ARG, "%s: %lld rows: at most 2^27 - 1", what, (long long)M);
  WANMI_REQUIRE(K >= 16 && K % 16 == 0 && K < (1 << 22), WANMI_ERR_ARG, "%s: K=%lld must be a multiple of 16 below 2^22", what, (long long)K);
  return WANMI_OK;
}

}  // namespace wanmi

extern "C" int wanmi_fp8_block_quantize(const void* x, int64_t ldx, int64_t M, int64_t K, uint8_t* codes, float* scales, int64_t s_row,
                                        int64_t s_blk, void* stream) {
  using namespace wanmi;
  clear_error();
  const char* what = "wanmi_fp8_block_quantize";
  const int bad = check_sizes(M, K, what);
  if (bad != WANMI_OK || M == 0) return bad;
  WANMI_REQUIRE(x && codes && scales, WANMI_ERR_ARG, "%s: null pointer", what);
  WANMI_REQUIRE((M == 1 || ldx >= K) && ldx % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)codes % 16 == 0, WANMI_ERR_ARG,
                "%s: rows of x (%lld apart) and the codes must be 16-byte aligned", what, (long long)ldx);
  // (a launch has fewer than 2^32 lanes)
  WANMI_REQUIRE(M * ((blocks_of(K) + 3) / 4) < (1LL << 26) - 4, WANMI_ERR_ARG, "%s: %lld x %lld is too large", what, (long long)M, (long long)K);
  launch_quantize((const uint16_t*)x, ldx, (int)M, (int)K, codes, scales, s_row, s_blk, (hipStream_t)stream);
  return check_launch(what);
}

namespace wanmi {

// The workspace: codes and scales of bf16 rows, or scales alone laid out block by block; then the parts of the sum.
struct Fp8Workspace {
  int64_t scales_at, parts_at, bytes;
  Fp8Plan plan;
};

static Fp8Workspace workspace_of(int64_t M, int64_t N, int64_t K, bool is_bf16, int64_t xs_row) {
  Fp8Workspace w{0, 0, 0, {kFp8Tiles256, 1, 0}};
  if (M <= 0 || N <= 0 || K <= 0 || M <= (is_bf16 ? kFewQuantize : kFewRows)) return w;
  auto round_up = [](int64_t n) { return (n + 255) / 256 * 256; };
  w.scales_at = is_bf16 ? round_up(M * K) : 0;
  w.bytes = w.parts_at = w.scales_at + (is_bf16 || xs_row != 1 ? round_up(M * blocks_of(K) * 4) : 0);
  if (M > kFewRows) {
    w.plan = fp8_plan(M, N, blocks_of(K));
    if (w.plan.splits > 1) w.bytes += w.plan.splits * M * N * 4;
  }
  return w;
}

}  // namespace wanmi

extern "C" int64_t wanmi_fp8_block_workspace(int64_t M, int64_t N, int64_t K, int is_bf16, int64_t xs_row) {
  return wanmi::workspace_of(M, N, K, is_bf16, xs_row).bytes;
}

extern "C" int wanmi_fp8_block_linear(const void* x, const float* x_scales, int64_t ldx, int64_t xs_row, int64_t xs_blk, const uint8_t* w,
                                      const float* w_scales, const float* bias, int64_t M, int64_t N, int64_t K, int gelu, void* out,
                                      int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace wanmi;
  clear_error();
  const char* what = "wanmi_fp8_block_linear";
  const int bad = check_sizes(M, K, what);
  if (bad != WANMI_OK) return bad;
  WANMI_REQUIRE(N >= 8 && N % 8 == 0 && N < (1 << 24), WANMI_ERR_ARG, "%s: N=%lld must be a multiple of 8 below 2^24", what, (long long)N);
  if (M == 0) return WANMI_OK;
  const bool is_bf16 = x_scales == nullptr;
  const int64_t KB = blocks_of(K), align = is_bf16 ? 8 : 16;
  WANMI_REQUIRE(x && w && w_scales && out, WANMI_ERR_ARG, "%s: null pointer", what);
  WANMI_REQUIRE(((uintptr_t)x | (uintptr_t)w | (uintptr_t)out | (uintptr_t)bias) % 16 == 0, WANMI_ERR_ARG, "%s: x, w, bias and out must be 16-byte aligned", what);
  WANMI_REQUIRE(ldx % align == 0 && (M == 1 || ldx >= K) && ldx < (1 << 23), WANMI_ERR_ARG, "%s: rows of x, %lld apart, must be 16-byte aligned", what, (long long)ldx);
  WANMI_REQUIRE(ldo % 8 == 0 && ldo >= N && ldo < (1 << 24), WANMI_ERR_ARG, "%s: the output's row stride %lld must be a multiple of 8 of at least N, below 2^24", what, (long long)ldo);
  const Fp8Workspace ws = workspace_of(M, N, K, is_bf16, xs_row);
  const int64_t need = ws.bytes;
  WANMI_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace && (uintptr_t)workspace % 16 == 0)), WANMI_ERR_ARG,
                "%s: the workspace holds %lld bytes of %lld", what, (long long)workspace_bytes, (long long)need);
  WANMI_REQUIRE(((M + 63) / 64) * ((N + 63) / 64) * ws.plan.splits < (1LL << 24) && M * ((KB + 3) / 4) < (1LL << 26) - 4, WANMI_ERR_ARG,
                "%s: %lld x %lld x %lld is too large for a launch", what, (long long)M, (long long)N, (long long)K);
  hipStream_t st = (hipStream_t)stream;
  Fp8Args g{(const uint8_t*)x, ldx, x_scales, xs_row, xs_blk, nullptr, w, w_scales, bias, (uint16_t*)out, ldo, (int)M, (int)N, (int)K, (int)KB, gelu, 0, 0, 1, nullptr};
  if (is_bf16 && M <= kFewQuantize) {
    g.x = (const uint16_t*)x;
  } else if (is_bf16) {
    uint8_t* codes = (uint8_t*)workspace;
    float* scales = (float*)(codes + ws.scales_at);
    launch_quantize((const uint16_t*)x, ldx, (int)M, (int)K, codes, scales, 1, M, st);
    g.a = codes, g.lda = K, g.a_scales = scales, g.as_row = 1, g.as_blk = M;
  } else if (M > kFewRows && xs_row != 1) {
    float* scales = (float*)workspace;
    hipLaunchKernelGGL(fp8_scales_kernel, dim3((unsigned)((M + 63) / 64)), dim3(256), 0, st, x_scales, xs_row, xs_blk, (int)M, (int)KB, scales);
    g.a_scales = scales, g.as_row = 1, g.as_blk = M;
  }
  if (M <= kFewRows) {
    const dim3 grid((unsigned)((N + 15) / 16)), block(64 * kFewWaves);
    if (g.x) hipLaunchKernelGGL((fp8_block_few_kernel<true>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((fp8_block_few_kernel<false>), grid, block, 0, st, g);
  } else {
    const int cus = device_cu_count();
    g.splits = ws.plan.splits;
    g.parts = (float*)((uint8_t*)workspace + ws.parts_at);
    switch (ws.plan.tiles) {
      case kFp8Tiles64: launch_tiles<64, 64, 2, 2, 4>(g, 0, st); break;
      case kFp8Tiles128Deep: launch_tiles<128, 128, 2, 4, 4>(g, 0, st); break;
      case kFp8Tiles128: launch_tiles<128, 128, 2, 4, 2>(g, 2 * cus, st); break;
      case kFp8Tiles256: launch_tiles<256, 256, 2, 4, 2>(g, cus, st); break;
    }
  }
  return check_launch(what);
}
