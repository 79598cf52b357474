// Low-rank adapters of many requests beside a shared projection (gfx950).
//
//   out[t, n] = bf16( base[t, n] + sum_j B[e][n, j] u[t, p(n) r + j] ),
//   u[t, i]   = scale[e] * row_scale[t] * sum_k A[e][i, k] x[t, k]
//
// e the adapter of row t's request (none: the row keeps its base), p(n) the part of a fused projection that column n
// belongs to; every part has r rows of A of its own. x is bf16 or MX codes with their block scales.
//
// Two launches: `shrink` forms u (fp32, in a workspace the caller owns), `expand` the rest. Which adapter a row
// uses is read on the GPU, row by row: a workgroup takes a tile of rows as they lie and goes through the distinct
// adapters it finds there (one, except where requests meet or are shorter than the tile), keeping of each
// product the columns of its own rows. Nothing has to be sorted or planned on the host, and a captured
// graph can be replayed with other ids. A row's product is a column of the MFMA of its own, so what
// lies in other rows, Inf and NaN too, does not reach it.
//
// Precision: x and A enter the MFMA as they are (an MX code times its scale is exact in bf16), u stays fp32, and the
// second product takes it as the sum of two bf16 values (u to 2^-16): an error of 2^-8 per rank would be
// as large as the output's own rounding where the adapter outweighs the base.
//
// The MFMA's rows are ranks (shrink) and output columns (expand), its columns tokens, so that a lane ends with
// consecutive ranks or columns of one token. The order of k inside a product is free as long as both
// operands agree: a lane takes consecutive k for all the MFMAs of a chunk, whole 16-byte pieces of codes.
#include <type_traits>

#include "wanmi_common.h"

namespace wanmi {
namespace {

constexpr int kMaxParts = 8;

struct LoraArgs {
  const void* x;
  const uint8_t* x_scales;  // null: x is bf16
  const float* row_scale;
  int64_t ldx;  // elements
  int64_t ldxs;
  const uint16_t* A;  // [adapters][parts * r][K]
  const uint16_t* B;  // [adapters][N][r]
  const float* scales;
  const int32_t* adapter_ids;
  const int32_t* request_ids;
  int requests, adapters;
  int64_t T;
  int K, N, r, R;  // R = parts * r
  int parts;
  int part_end[kMaxParts];
  int part_blocks[kMaxParts];  // workgroups of `span` columns
  int span;
  int splits, chunks_per_split, slots;
  int in_place;
  float* u;  // [splits][T][R]
  const uint16_t* base;
  int64_t ldb;
  uint16_t* out;
  int64_t ldo;
  int zero_rest;
};

// The adapter of row t: -1 none (the row keeps its base), -2 no request (the row is not computed).
__device__ __forceinline__ int row_adapter(const LoraArgs& a, int64_t t) {
  if (t >= a.T) return -2;
  const int q = a.request_ids ? a.request_ids[t] : (int)t;
  if ((uint32_t)q >= (uint32_t)a.requests) return -2;  // (adapter_ids ends there)
  const int e = a.adapter_ids[q];
  return (uint32_t)e < (uint32_t)a.adapters ? e : -1;
}

// The smallest adapter above `prev` among the rows of a tile (v0, v1: the lane's rows'), INT_MAX if there is none.
__device__ __forceinline__ int next_adapter(int v0, int v1, int prev) {
  int v = min(v0 > prev ? v0 : 0x7FFFFFFF, v1 > prev ? v1 : 0x7FFFFFFF);
  v = min(v, dpp_i32<0xB1>(v));
  v = min(v, dpp_i32<0x4E>(v));
  v = min(v, dpp_i32<0x141>(v));
  v = min(v, dpp_i32<0x140>(v));
#pragma unroll
  for (int o = 16; o <= 32; o <<= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// Eight MX codes (two words) times their block's scale -> bf16, exact.
__device__ __forceinline__ bf16x8 mx_to_bf16(uint32_t w0, uint32_t w1, float scale) {
  union { bf16x8 v; bf16x2_t p[4]; } f;
  f.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  f.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  f.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  f.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return f.v;
}

// ------------------------------------------------------------------------------------------------
// shrink, few rows: 32 rows x 64 ranks a workgroup, K split over its four waves and over workgroups
// ------------------------------------------------------------------------------------------------
// A's rows are what has to be read here: every lane loads its 64 bytes of a chunk of 128 k straight
// into the MFMA's layout. blockIdx.z counts splits of K and, where a tile may hold several adapters, slots:
// slot s takes the adapters s, s + slots, ... that the tile's rows use.
constexpr int kRows = 32;
constexpr int kRankTiles = 4;

template <bool kMx>
__global__ __launch_bounds__(256) void lora_shrink_few_kernel(LoraArgs a) {
  __shared__ f32x4 red[4][2 * kRankTiles][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t t0 = (int64_t)blockIdx.x * kRows;
  const int rank0 = blockIdx.y * 16 * kRankTiles;
  const int split = blockIdx.z % a.splits, slot = blockIdx.z / a.splits;
  const int nchunks = (a.K + 127) / 128;
  const int ch0 = split * a.chunks_per_split, ch1 = min(ch0 + a.chunks_per_split, nchunks);
  const int mine = lane < kRows ? row_adapter(a, t0 + lane) : -2;
  int64_t row[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) row[m] = min(t0 + 16 * m + c, a.T - 1);  // rows past the end: loaded again, not used
  int e = -1;
  for (int at = 0;; ++at) {
    e = next_adapter(mine, -2, e);
    if (e == 0x7FFFFFFF) break;
    if (at % a.slots != slot) continue;
    const uint64_t match = __ballot(mine == e);
    f32x4 acc[2][kRankTiles];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int rt = 0; rt < kRankTiles; ++rt) acc[m][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint16_t* pa = a.A + ((int64_t)e * a.R + rank0 + c) * a.K;
    for (int ch = ch0 + wave; ch < ch1; ch += 4) {
      const int k = ch * 128 + 32 * g;
      const bool in = k < a.K;
      bf16x8 xf[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        if (kMx) {
          u32x4 w[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
          float sc = 0.0f;
          if (in) {
            const u32x4* px = reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(a.x) + row[m] * a.ldx + k);
            w[0] = px[0];
            w[1] = px[1];
            sc = __uint_as_float((uint32_t)a.x_scales[row[m] * a.ldxs + (k >> 5)] << 23);
          }
#pragma unroll
          for (int s = 0; s < 4; ++s) xf[m][s] = mx_to_bf16(w[s >> 1][2 * (s & 1)], w[s >> 1][2 * (s & 1) + 1], sc);
        } else {
          const u32x4* px = reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(a.x) + row[m] * a.ldx + k);
#pragma unroll
          for (int s = 0; s < 4; ++s) xf[m][s] = __builtin_bit_cast(bf16x8, in ? px[s] : u32x4{0u, 0u, 0u, 0u});
        }
      }
#pragma unroll
      for (int rt = 0; rt < kRankTiles; ++rt) {
        if (rank0 + 16 * rt < a.R) {
          const u32x4* pw = reinterpret_cast<const u32x4*>(pa + (int64_t)16 * rt * a.K + k);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const bf16x8 af = __builtin_bit_cast(bf16x8, in ? pw[s] : u32x4{0u, 0u, 0u, 0u});
#pragma unroll
            for (int m = 0; m < 2; ++m) acc[m][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, xf[m][s], acc[m][rt], 0, 0, 0);
          }
        }
      }
    }
    // the four waves' partial sums, added in the waves' order; wave w finishes two of the eight tiles
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int rt = 0; rt < kRankTiles; ++rt) red[wave][m * kRankTiles + rt][lane] = acc[m][rt];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int tile = 2 * wave + i, m = tile / kRankTiles, rt = tile % kRankTiles;
      f32x4 v = red[0][tile][lane];
#pragma unroll
      for (int w = 1; w < 4; ++w) v += red[w][tile][lane];
      const int rank = rank0 + 16 * rt + 4 * g;
      if (rank < a.R && (match >> (16 * m + c) & 1)) {
        float f = a.scales ? a.scales[e] : 1.0f;
        if (a.row_scale) f *= a.row_scale[row[m]];
        v *= f;
        *reinterpret_cast<f32x4*>(a.u + ((int64_t)split * a.T + row[m]) * a.R + rank) = v;
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------
// shrink, many rows: 256 rows x 128 ranks a workgroup of eight waves, or 128 rows x 64 or 32 ranks of four
// ------------------------------------------------------------------------------------------------
// Both operands pass through LDS, loaded straight into it (16-byte pieces, whole 128-byte runs of a row per
// eight lanes), in rings of three: A by steps of 64 k, x by 128 bytes of a row (64 k, or 128 of MX codes). x is read
// once per kNR ranks and A once per tile of rows. A wave's tile is 64 rows x 64 ranks at kNR = 128, where its operand
// reads from LDS take less time than its MFMAs, and 32 rows x kNR ranks below, where x is what there is to read and
// two workgroups a CU keep more of it under way. Piece p of row i lies in slot p ^ (i & 7) of the row, so that the
// eight rows that are read together take different banks. The MX scales come with x, four bytes per row.
// 32768 rows of one request, MX: K = 5120, 32 ranks 58 us and 64 ranks 63 (x alone at 5.5 TB/s: 32; 64 rows of x at
// a time come in runs of 128 bytes, and neither longer runs nor another order of k brought more than 3 TB/s), K =
// 13824, 128 ranks 154 (753 TFLOP/s).
// Where requests meet inside a tile, each adapter takes a sweep over K of its own, in which the waves without rows
// of it only load. The sweeps are shared out over two workgroups (slots; the second one ends at once where a tile
// has one adapter), so that they run side by side where the chip has room: QKV of 7799 rows in 5 requests, 4
// adapters, rank 64: 42 us, one workgroup for all of a tile's sweeps 56; K = 13824, 32760 rows in 3 requests, rank 128: 141
// and 230.
template <bool kMx, int kNR>
struct Big {
  static constexpr int kWaves = kNR == 128 ? 8 : 4;
  static constexpr int kRows = 32 * kWaves;
  static constexpr int kX = kRows * 128;  // bytes of a stage
  static constexpr int kA = kNR * 128;
  static constexpr int kScales = kMx ? 3 * kRows * 4 : 0;
  static constexpr int kLds = 3 * (kX + kA) + kScales;
  static constexpr int kXLoads = 4 + (kMx ? 1 : 0), kALoads = kA / 1024 / kWaves;  // per wave
  static constexpr int kMT = kNR == 128 ? 4 : 2;  // the wave's tile: 16 kMT rows, 16 kRT ranks
  static constexpr int kRT = kNR == 128 ? 4 : kNR / 16;
};

template <bool kMx, int kNR>
__global__ __launch_bounds__(kNR == 128 ? 512 : 256, 2) void lora_shrink_kernel(LoraArgs a) {
  using P = Big<kMx, kNR>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t t0 = (int64_t)blockIdx.x * P::kRows;
  const int rank0 = blockIdx.y * kNR;
  const int rows = (int)min((int64_t)P::kRows, a.T - t0);
  const int nranks = min(kNR, a.R - rank0);
  const int m0 = (kNR == 128 ? wave >> 1 : wave) * 16 * P::kMT;  // the wave's first row and rank
  const int r0 = kNR == 128 ? (wave & 1) * 64 : 0;
  const int split = blockIdx.z % a.splits, slot = blockIdx.z / a.splits;
  const int ch0 = split * a.chunks_per_split, n = min(a.chunks_per_split, a.K / 64 - ch0);  // (even for MX)

  int v[P::kRows / 64];  // the tile's adapters
#pragma unroll
  for (int i = 0; i < P::kRows / 64; ++i) v[i] = row_adapter(a, t0 + 64 * i + lane);

  constexpr int xes = kMx ? 1 : 2;
  const uint8_t* xb = reinterpret_cast<const uint8_t*>(a.x) + (t0 * a.ldx + (int64_t)ch0 * 64) * xes;
  const u32x4 rx = buffer_rsrc(xb, (uint32_t)(((int64_t)(rows - 1) * a.ldx + (int64_t)n * 64) * xes));  // rows past the end: zeros
  u32x4 rs = {0u, 0u, 0u, 0u};
  if (kMx) rs = buffer_rsrc(a.x_scales + t0 * a.ldxs + ch0 * 2, (uint32_t)((rows - 1) * a.ldxs + n * 2));
  // Lane offsets of the loads, eight rows to an instruction: everything that does not change with the step is in
  // them, and the step's own part is a scalar (within a row, so never past an extent by itself).
  const int li = lane >> 3;
  const uint32_t lp = (uint32_t)(((lane & 7) ^ li) << 4);
  uint32_t xo[4], ao[P::kALoads];
#pragma unroll
  for (int j = 0; j < 4; ++j) xo[j] = (uint32_t)((8 * (P::kWaves * j + wave) + li) * a.ldx * xes) + lp;
#pragma unroll
  for (int j = 0; j < P::kALoads; ++j) ao[j] = (uint32_t)((8 * (P::kWaves * j + wave) + li) * a.K * 2) + lp;
  // (the upper half of the waves loads the same scales again: equal counts in every wave)
  const uint32_t so = (uint32_t)((64 * (wave % (P::kWaves / 2)) + lane) * a.ldxs);
  const uint32_t base = lds_addr(lds);
  constexpr int kAAt = 3 * P::kX, kSAt = 3 * (P::kX + P::kA);
  constexpr int kXSteps = kMx ? 2 : 1;  // steps of 64 k to a stage of x
  // and of the reads, for the two halves of a step (A, bf16 x) or of a stage (codes)
  const uint8_t* xr = lds + (m0 + c) * 128;
  const uint8_t* ar = lds + kAAt + (r0 + c) * 128;
  const int half[2] = {((2 * g) ^ (c & 7)) << 4, ((2 * g + 1) ^ (c & 7)) << 4};
  const int xhalf[2] = {kMx ? (g ^ (c & 7)) << 4 : half[0], kMx ? ((4 + g) ^ (c & 7)) << 4 : half[1]};
  const uint8_t* sr = lds + kSAt + (m0 + c) * 4 + (g >> 1);

  int e = -1;
  for (int at = 0;; ++at) {
    int next = next_adapter(v[0], v[1], e);
    if (P::kRows > 128) next = min(next, next_adapter(v[P::kRows / 64 - 2], v[P::kRows / 64 - 1], e));
    e = next;
    if (e == 0x7FFFFFFF) break;
    if (at % a.slots != slot) continue;
    uint64_t here = 0;
#pragma unroll
    for (int i = 0; i < P::kRows / 64; ++i) {
      const uint64_t b = __ballot(v[i] == e);
      if (m0 / 64 == i) here = b >> (m0 & 63);
    }
    const bool mine = (P::kMT == 4 ? here : here & 0xFFFFFFFFu) != 0;
    const u32x4 ra = buffer_rsrc(a.A + ((int64_t)e * a.R + rank0) * a.K + ch0 * 64,
                                 (uint32_t)(((int64_t)(nranks - 1) * a.K + (int64_t)n * 64) * 2));  // ranks past the end: zeros
    const auto issue_x = [&](int i, int slot) {
#pragma unroll
      for (int j = 0; j < 4; ++j) lds_dma_b128(rx, xo[j], (uint32_t)(i * 128), base + slot * P::kX + (P::kWaves * j + wave) * 1024);
      if (kMx) lds_dma_b32(rs, so, (uint32_t)(i * 4), base + kSAt + slot * (P::kRows * 4) + wave % (P::kWaves / 2) * 256);
    };
    const auto issue_a = [&](int i, int slot) {
#pragma unroll
      for (int j = 0; j < P::kALoads; ++j)
        lds_dma_b128(ra, ao[j], (uint32_t)(i * 128), base + kAAt + slot * P::kA + (P::kWaves * j + wave) * 1024);
    };
    f32x4 acc[P::kMT][P::kRT];
#pragma unroll
    for (int m = 0; m < P::kMT; ++m)
#pragma unroll
      for (int rt = 0; rt < P::kRT; ++rt) acc[m][rt] = f32x4{0.f, 0.f, 0.f, 0.f};
    // the adapter before: its stores are out of the count below, and the stages' last readers are done
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    __syncthreads();
    issue_x(0, 0);
    issue_a(0, 0);
    if (kXSteps < n) issue_x(1, 1);
    if (n > 1) issue_a(1, 1);
    // Step i of the rings' period of six (J = i % 6): every place in LDS is a constant.
    const auto step = [&](auto J, int i) {
      constexpr int j = decltype(J)::value, as = j % 3, xs = j / kXSteps % 3, h = j % kXSteps;
      // Step i issues A's stage i + 2 and, every kXSteps, x's stage two ahead: behind the loads of step i, this wave
      // has issued one stage of each when it gets here.
      if (i + 3 >= n) __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      else __builtin_amdgcn_s_waitcnt(waitcnt_vm(P::kXLoads + P::kALoads));
      __syncthreads();
      if (i + 2 < n) issue_a(i + 2, (as + 2) % 3);
      if (h == 0 && i + 2 * kXSteps < n) issue_x(i / kXSteps + 2, (xs + 2) % 3);
      if (!mine) return;
      // the codes of one row group are converted while the MFMAs of the one before run
      u32x4 xw[P::kMT][kMx ? 1 : 2];
      float sc[P::kMT];
#pragma unroll
      for (int m = 0; m < P::kMT; ++m) {
        if (kMx) {
          xw[m][0] = *reinterpret_cast<const u32x4*>(xr + xhalf[h] + xs * P::kX + m * 2048);
          sc[m] = __uint_as_float((uint32_t)sr[xs * (P::kRows * 4) + m * 64 + 2 * h] << 23);
        } else {
#pragma unroll
          for (int s = 0; s < 2; ++s) xw[m][kMx ? 0 : s] = *reinterpret_cast<const u32x4*>(xr + xhalf[s] + xs * P::kX + m * 2048);
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf16x8 af[P::kRT];
#pragma unroll
        for (int rt = 0; rt < P::kRT; ++rt) af[rt] = *reinterpret_cast<const bf16x8*>(ar + half[s] + as * P::kA + rt * 2048);
#pragma unroll
        for (int m = 0; m < P::kMT; ++m) {
          const bf16x8 xf = kMx ? mx_to_bf16(xw[m][0][2 * s], xw[m][0][2 * s + 1], sc[m]) : __builtin_bit_cast(bf16x8, xw[m][kMx ? 0 : s]);
#pragma unroll
          for (int rt = 0; rt < P::kRT; ++rt) acc[m][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[rt], xf, acc[m][rt], 0, 0, 0);
        }
      }
    };
    for (int i = 0;;) {
      step(std::integral_constant<int, 0>{}, i);
      if (++i == n) break;
      step(std::integral_constant<int, 1>{}, i);
      if (++i == n) break;
      step(std::integral_constant<int, 2>{}, i);
      if (++i == n) break;
      step(std::integral_constant<int, 3>{}, i);
      if (++i == n) break;
      step(std::integral_constant<int, 4>{}, i);
      if (++i == n) break;
      step(std::integral_constant<int, 5>{}, i);
      if (++i == n) break;
    }
    const float se = a.scales ? a.scales[e] : 1.0f;
#pragma unroll
    for (int m = 0; m < P::kMT; ++m) {
      const int64_t t = t0 + m0 + 16 * m + c;
      if (row_adapter(a, t) != e) continue;
      const float f = a.row_scale ? se * a.row_scale[t] : se;
#pragma unroll
      for (int rt = 0; rt < P::kRT; ++rt) {
        const int rank = r0 + 16 * rt + 4 * g;
        if (rank < nranks) *reinterpret_cast<f32x4*>(a.u + ((int64_t)split * a.T + t) * a.R + rank0 + rank) = acc[m][rt] * f;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// expand: 16 kRG rows x up to `span` columns of one part a workgroup
// ------------------------------------------------------------------------------------------------
// The rows' u are added over the splits of K and laid in LDS as the MFMA's operand, high and low bf16 halves, once;
// then each wave takes blocks of 64 columns: B's fragments once (in registers for kKS steps of 32 ranks; kKS = 0:
// any rank, read again for every pair of row groups), the rows in groups of 16, the base of the next group
// under way while the MFMAs of this one run.
// Row i of MFMA operand tile s stands for column 32 (s / 2) + 8 (i / 4) + 4 (s % 2) + i % 4 of the block: a lane
// ends with two runs of 8 consecutive columns, and the lanes of a row cover 64 bytes at a time.
template <int kRG, int kKS>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  __shared__ int sad[kRG * 16];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t t0 = (int64_t)blockIdx.x * (16 * kRG);
  const int slot = blockIdx.z;
  int part = 0, blk = blockIdx.y;
  while (blk >= a.part_blocks[part]) blk -= a.part_blocks[part++];
  const int pend = a.part_end[part];
  const int col0 = (part ? a.part_end[part - 1] : 0) + blk * a.span;
  const int col1 = min(col0 + a.span, pend);
  const int ks = kKS > 0 ? kKS : (a.r + 31) / 32;

  if (threadIdx.x < kRG * 16) sad[threadIdx.x] = row_adapter(a, t0 + threadIdx.x);
  u32x4* frag = reinterpret_cast<u32x4*>(lds);  // [row group][step][high, low][lane]
  for (int i = threadIdx.x; i < kRG * 16 * ks * 4; i += 256) {
    const int row = i / (ks * 4), piece = i % (ks * 4);
    const int64_t t = t0 + row;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.0f;
    if (t < a.T && piece * 8 < a.r) {  // (rows without an adapter: whatever lies there, not used)
      const float* pu = a.u + t * a.R + part * a.r + piece * 8;
#pragma unroll 4
      for (int q = 0; q < a.splits; ++q) {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(pu + q * a.T * a.R), hi = *reinterpret_cast<const f32x4*>(pu + q * a.T * a.R + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] += lo[j], f[4 + j] += hi[j];
      }
    }
    // u = uh + ul; an infinity is uh alone
    u32x4 uh, ul;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uh[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
      const float h0 = bf16_lo(uh[j]), h1 = bf16_hi(uh[j]);
      ul[j] = pack_bf16x2(fabsf(h0) < INFINITY ? f[2 * j] - h0 : 0.0f, fabsf(h1) < INFINITY ? f[2 * j + 1] - h1 : 0.0f);
    }
    u32x4* to = frag + ((row >> 4) * ks + (piece >> 2)) * 128 + (piece & 3) * 16 + (row & 15);
    to[0] = uh;
    to[64] = ul;
  }
  __syncthreads();
  const int v0 = lane < kRG * 16 ? sad[lane] : -2, v1 = lane + 64 < kRG * 16 ? sad[lane + 64] : -2;
  int ad[kRG];
#pragma unroll
  for (int m = 0; m < kRG; ++m) ad[m] = sad[16 * m + c];

  int e = next_adapter(v0, v1, -1);
  for (int at = 0; at == 0 || e != 0x7FFFFFFF; ++at, e = next_adapter(v0, v1, e)) {
    if (at % a.slots != slot) continue;
    const bool product = e != 0x7FFFFFFF;
    // the rows of this pass: those of adapter e, and in the first one those that only keep their base or become zero
    bool take[kRG];
#pragma unroll
    for (int m = 0; m < kRG; ++m)
      take[m] = t0 + 16 * m + c < a.T && ((product && ad[m] == e) || (at == 0 && ((ad[m] == -1 && !a.in_place) || (ad[m] == -2 && a.zero_rest))));
    for (int n0 = col0 + 64 * wave; n0 < col1; n0 += 256) {
      const int nl = n0 + 8 * g;  // the lane's columns: nl .. nl + 7 and 32 on
      const bool ok[2] = {nl + 8 <= pend, nl + 40 <= pend};
      const auto brow = [&](int s) {
        const int n = min(n0 + 32 * (s >> 1) + 8 * (c >> 2) + 4 * (s & 1) + (c & 3), pend - 1);
        return a.B + ((int64_t)e * a.N + n) * a.r + 8 * g;
      };
      const auto load_base = [&](int m, u32x4 (&o)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          o[h] = u32x4{0u, 0u, 0u, 0u};
          if (take[m] && ad[m] != -2 && ok[h]) o[h] = *reinterpret_cast<const u32x4*>(a.base + (t0 + 16 * m + c) * a.ldb + nl + 32 * h);
        }
      };
      const auto finish = [&](int m, u32x4 (&o)[2], const f32x4 (&acc)[4]) {
        if (ad[m] >= 0) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              o[h][j] = pack_bf16x2(bf16_lo(o[h][j]) + acc[2 * h + j / 2][2 * (j & 1)],
                                    bf16_hi(o[h][j]) + acc[2 * h + j / 2][2 * (j & 1) + 1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (take[m] && ok[h]) store_b128_guarded(o[h], a.out + (t0 + 16 * m + c) * a.ldo + nl + 32 * h);
      };
      if constexpr (kKS > 0) {
        bf16x8 bf[kKS][4];
        if (product) {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const uint16_t* pb = brow(s);
#pragma unroll
            for (int k = 0; k < kKS; ++k)
              bf[k][s] = __builtin_bit_cast(bf16x8, 32 * k + 8 * g < a.r ? *reinterpret_cast<const u32x4*>(pb + 32 * k) : u32x4{0u, 0u, 0u, 0u});
          }
        } else {
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int k = 0; k < kKS; ++k) bf[k][s] = __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
        }
        u32x4 cur[2], nxt[2];
        load_base(0, cur);
#pragma unroll
        for (int m = 0; m < kRG; ++m) {
          if (m + 1 < kRG) load_base(m + 1, nxt);
          f32x4 acc[4];
#pragma unroll
          for (int s = 0; s < 4; ++s) acc[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < kKS; ++k) {
            const bf16x8 uh = __builtin_bit_cast(bf16x8, frag[(m * kKS + k) * 128 + lane]);
            const bf16x8 ul = __builtin_bit_cast(bf16x8, frag[(m * kKS + k) * 128 + 64 + lane]);
#pragma unroll
            for (int s = 0; s < 4; ++s) acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[k][s], uh, acc[s], 0, 0, 0);
#pragma unroll
            for (int s = 0; s < 4; ++s) acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[k][s], ul, acc[s], 0, 0, 0);
          }
          finish(m, cur, acc);
#pragma unroll
          for (int h = 0; h < 2; ++h) cur[h] = nxt[h];
        }
      } else {
        u32x4 cur[kRG][2];
#pragma unroll
        for (int m = 0; m < kRG; ++m) load_base(m, cur[m]);
        f32x4 acc[kRG][4];
#pragma unroll
        for (int m = 0; m < kRG; ++m)
#pragma unroll
          for (int s = 0; s < 4; ++s) acc[m][s] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (product) {
          for (int k = 0; k < ks; ++k) {
            bf16x8 bf[4];
#pragma unroll
            for (int s = 0; s < 4; ++s)
              bf[s] = __builtin_bit_cast(bf16x8, 32 * k + 8 * g < a.r ? *reinterpret_cast<const u32x4*>(brow(s) + 32 * k) : u32x4{0u, 0u, 0u, 0u});
#pragma unroll
            for (int m = 0; m < kRG; ++m) {
              const bf16x8 uh = __builtin_bit_cast(bf16x8, frag[(m * ks + k) * 128 + lane]);
              const bf16x8 ul = __builtin_bit_cast(bf16x8, frag[(m * ks + k) * 128 + 64 + lane]);
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                acc[m][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[s], uh, acc[m][s], 0, 0, 0);
                acc[m][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[s], ul, acc[m][s], 0, 0, 0);
              }
            }
          }
        }
#pragma unroll
        for (int m = 0; m < kRG; ++m) finish(m, cur[m], acc[m]);
      }
    }
    if (!product) break;
  }
}

// ------------------------------------------------------------------------------------------------
// expand, many rows: 128 rows x `span` columns a workgroup, rank at most 32 kKS <= 128
// ------------------------------------------------------------------------------------------------
// A wave keeps u of its 32 rows in registers and walks the columns in blocks of 64; the block's rows of B go
// through LDS, shared by the four waves, two blocks ahead. base and out move as whole 128-byte runs of a
// row, eight rows to an instruction (lanes that are neighbours and not contiguous cost the texture unit an access
// each: in the MFMA's own layout these loads and stores took it 64 accesses instead of 16, and were the bound), so the
// sums pass through a piece of LDS of the wave's own on their way to that layout.
// Rows and columns that are not to be written have offsets past the descriptors' extents: every wave with rows
// of the pass issues the same loads and stores, and the waits below can count them.
template <int kKS>
struct Many {
  static constexpr int kPitch = 64 * kKS;  // bytes of a row of B in LDS
  static constexpr int kB = 64 * kPitch;
  static constexpr int kStages = 3;
  static constexpr int kLoads = kB / 4096;  // per wave and block
  static constexpr int kRow = 68;           // floats of a row of the wave's piece: 4 more than the block's columns
  static constexpr int kLds = kStages * kB + 4 * 16 * kRow * 4;
};

template <int kKS>
__global__ __launch_bounds__(256, 2) void lora_expand_many_kernel(LoraArgs a) {
  using P = Many<kKS>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t t0 = (int64_t)blockIdx.x * 128;
  int part = 0, blk = blockIdx.y;
  while (blk >= a.part_blocks[part]) blk -= a.part_blocks[part++];
  const int pend = a.part_end[part];
  const int col0 = (part ? a.part_end[part - 1] : 0) + blk * a.span;
  const int n = (min(a.span, pend - col0) + 63) / 64;

  const int v0 = row_adapter(a, t0 + lane), v1 = row_adapter(a, t0 + 64 + lane);
  int e = next_adapter(v0, v1, -1);
  // u of the wave's rows (two groups of 16) as the MFMA's operand: high and low halves. The splits of K are added two at a time
  // with all of their loads under way (4096 rows x 5120 columns, rank 32, four splits: 38.5 us a call, one by one 39.0).
  bf16x8 uh[2][kKS], ul[2][kKS];
  {
    float f[2][kKS][8];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int k = 0; k < kKS; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) f[m][k][j] = 0.0f;
    const float* pu[2];
#pragma unroll
    for (int m = 0; m < 2; ++m)  // (rows without an adapter: whatever lies there, not used)
      pu[m] = a.u + min(t0 + 32 * wave + 16 * m + c, a.T - 1) * a.R + part * a.r + 8 * g;
    for (int q = 0; q < a.splits; q += 2) {
      f32x4 w[2][2][kKS][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int k = 0; k < kKS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              w[h][m][k][i] = f32x4{0.f, 0.f, 0.f, 0.f};
              if (q + h < a.splits && 32 * k + 8 * g < a.r)
                w[h][m][k][i] = *reinterpret_cast<const f32x4*>(pu[m] + (q + h) * a.T * a.R + 32 * k + 4 * i);
            }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int k = 0; k < kKS; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) f[m][k][j] += w[h][m][k][j >> 2][j & 3];
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int k = 0; k < kKS; ++k) {
        u32x4 h, l;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = f[m][k][2 * j], y = f[m][k][2 * j + 1];
          h[j] = pack_bf16x2(x, y);
          const float h0 = bf16_lo(h[j]), h1 = bf16_hi(h[j]);
          l[j] = pack_bf16x2(fabsf(h0) < INFINITY ? x - h0 : 0.0f, fabsf(h1) < INFINITY ? y - h1 : 0.0f);
        }
        uh[m][k] = __builtin_bit_cast(bf16x8, h);
        ul[m][k] = __builtin_bit_cast(bf16x8, l);
      }
  }

  // the rows that this lane loads and stores: 16 m + 8 h + lane / 8 of the wave's, columns 8 (lane & 7) .. + 7
  const int rows = (int)min((int64_t)128, a.T - t0);
  const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.base + t0 * a.ldb), (short)0, (int)(((rows - 1) * a.ldb + a.N) * 2), 0x00020000);
  const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(a.out + t0 * a.ldo, (short)0, (int)(((rows - 1) * a.ldo + a.N) * 2), 0x00020000);
  constexpr uint32_t kNone = 0xFFFFFF00u;
  const int c8 = 8 * (lane & 7);
  int ad[4];
  uint32_t ob[4], oo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 32 * wave + 8 * i + (lane >> 3);
    ad[i] = __shfl(wave < 2 ? v0 : v1, row & 63, 64);
    ob[i] = (uint32_t)((row * a.ldb + col0 + c8) * 2);
    oo[i] = (uint32_t)((row * a.ldo + col0 + c8) * 2);
  }
  // a row of B's block is 4 kKS pieces of 16 bytes, each in the slot of that row that `swizzle` gives
  constexpr int kPieces = 4 * kKS, kRowsPer = 64 / kPieces;
  const int bi = lane / kPieces;
  const uint32_t ldsb = lds_addr(lds);
  float* piece = reinterpret_cast<float*>(lds + P::kStages * P::kB) + wave * 16 * P::kRow;
  const auto swizzle = [](int row) { return kKS == 1 ? (row >> 1) & 3 : row & (kPieces - 1); };

  for (int at = 0; at == 0 || e != 0x7FFFFFFF; ++at, e = next_adapter(v0, v1, e)) {
    const bool product = e != 0x7FFFFFFF;
    bool take[4], any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 32 * wave + 8 * i + (lane >> 3);
      take[i] = row < rows && ((product && ad[i] == e) || (at == 0 && ((ad[i] == -1 && !a.in_place) || (ad[i] == -2 && a.zero_rest))));
      any |= take[i];
    }
    const bool mine = __ballot(any) != 0;
    const u32x4 rB = buffer_rsrc(product ? a.B + ((int64_t)e * a.N + col0) * a.r : a.B, product ? (uint32_t)((pend - col0) * a.r * 2) : 0u);
    const auto issue = [&](int b) {
#pragma unroll
      for (int j = 0; j < P::kLoads; ++j) {
        const int row = kRowsPer * (4 * j + wave) + bi;
        const int pc = (lane % kPieces) ^ swizzle(row);
        lds_dma_b128(rB, 8 * pc < a.r ? (uint32_t)((64 * b + row) * a.r * 2 + 16 * pc) : kNone,
                     ldsb + (b % P::kStages) * P::kB + (4 * j + wave) * 1024);
      }
    };
    const auto load_base = [&](int b, u32x4 (&o)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = __builtin_amdgcn_raw_buffer_load_b128(
            rb, take[i] && ad[i] != -2 && col0 + 64 * b + c8 + 8 <= pend ? ob[i] + 128 * b : kNone, 0, 0);
    };
    if (at) {  // the adapter before: its stores are out of the counts below, and the stages' last readers are done
      __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      __syncthreads();
    }
    issue(0);
    if (n > 1) issue(1);
    u32x4 cur[4], nxt[4];
    if (mine) load_base(0, cur);
    for (int b = 0; b < n; ++b) {
      // This wave's loads of block b have arrived when only what it issued after them is under way: the base of the
      // blocks b - 1 and b, the stores of b - 2 and b - 1 (four each) and the next block of B.
      if (!mine) {
        if (b + 1 < n) __builtin_amdgcn_s_waitcnt(waitcnt_vm(P::kLoads));
        else __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      } else if (b + 1 >= n || b == 0) {
        if (b == 0 && b + 1 < n) __builtin_amdgcn_s_waitcnt(waitcnt_vm(4 + P::kLoads));
        else if (b == 0) __builtin_amdgcn_s_waitcnt(waitcnt_vm(4));
        else __builtin_amdgcn_s_waitcnt(waitcnt_vm(12));
      } else if (b == 1) {
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(12 + P::kLoads));
      } else {
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(16 + P::kLoads));
      }
      __syncthreads();
      if (b + 2 < n) issue(b + 2);
      if (!mine) continue;
      if (b + 1 < n) load_base(b + 1, nxt);
      const uint8_t* sb = lds + (b % P::kStages) * P::kB;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        f32x4 acc[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) acc[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kKS; ++k)
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int row = 16 * s + c;
            const bf16x8 bf = *reinterpret_cast<const bf16x8*>(sb + row * P::kPitch + (((4 * k + g) ^ swizzle(row)) << 4));
            acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf, uh[m][k], acc[s], 0, 0, 0);
            acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf, ul[m][k], acc[s], 0, 0, 0);
          }
#pragma unroll
        for (int s = 0; s < 4; ++s) *reinterpret_cast<f32x4*>(piece + c * P::kRow + 16 * s + 4 * g) = acc[s];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = 2 * m + h;
          const f32x4 d0 = *reinterpret_cast<const f32x4*>(piece + (8 * h + (lane >> 3)) * P::kRow + c8);
          const f32x4 d1 = *reinterpret_cast<const f32x4*>(piece + (8 * h + (lane >> 3)) * P::kRow + c8 + 4);
          u32x4 o = cur[i];
          if (ad[i] >= 0) {
            o[0] = pack_bf16x2(bf16_lo(o[0]) + d0[0], bf16_hi(o[0]) + d0[1]);
            o[1] = pack_bf16x2(bf16_lo(o[1]) + d0[2], bf16_hi(o[1]) + d0[3]);
            o[2] = pack_bf16x2(bf16_lo(o[2]) + d1[0], bf16_hi(o[2]) + d1[1]);
            o[3] = pack_bf16x2(bf16_lo(o[3]) + d1[2], bf16_hi(o[3]) + d1[3]);
          }
          store_b128_guarded(o, ro, take[i] && col0 + 64 * b + c8 + 8 <= pend ? oo[i] + 128 * b : kNone, 0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) cur[i] = nxt[i];
    }
    if (!product) break;
  }
}

// Which kernels a call takes. Many rows take the large tiles: below 1024 rows there are too few of them
// to fill the chip. Whole calls in us, N = 5120, small tiles / large tiles, MX:
//   rows                                          512         1024        2048        4096
//   K =  5120, rank  16,  1 adapter            10.9 / 16.8 15.2 / 20.1 19.8 / 23.2 30.1 / 28.8
//   K =  5120, rank  32,  8 adapters           16.3 / 21.8 21.2 / 23.4 29.7 / 25.5 42.7 / 32.4
//   K =  5120, rank  64,  4 adapters           19.4 / 26.1 28.7 / 31.2 37.6 / 33.8 56.0 / 40.5
//   K = 13824, rank 128,  1 adapter            29.1 / 70.3 42.0 / 82.0 66.6 / 86.1 118  / 111
// So from 1024 rows to the crossing (2048, at one adapter 3000 to 4000) the small tiles would do as well or better,
// most of all at rank 128; the bound is the number of rows alone.
// K that is no multiple of 128 is left to the small tiles, as are rows past the large ones' 32-bit offsets: their
// rows of A come from L2 again for every 32 rows. 32760 rows, MX, K = 5088 against 5120: rank 16 221 / 186 us, 32 243 /
// 188, 64 275 / 194, 128 349 / 225 (4096 rows: 29 / 29, 34 / 32, 44 / 39, 66 / 78; K = 1504 against 1536 at 32760: 166 / 159 to
// 214 / 190).
// The chip's 256 CUs are constants here: the caller sizes the workspace by the same plan, on whichever device is current.
struct LoraPlan {
  bool big;
  int nr;  // ranks of a workgroup (big)
  int splits, chunks_per_split, slots;
};

// `plain`: whether x allows the tiles' loads.
LoraPlan lora_plan(int64_t T, int64_t K, int64_t R, int64_t adapters, bool plain) {
  LoraPlan p{};
  p.big = plain && T >= 1024 && K % 128 == 0 && K < (1LL << 21);
  p.slots = 1;
  if (p.big) {
    p.nr = R <= 32 ? 32 : R % 128 == 0 ? 128 : 64;
    const int64_t rows = p.nr == 128 ? 256 : 128, resident = p.nr == 128 ? 256 : 512;  // on 256 CUs
    const int64_t wgs = (T + rows - 1) / rows * ((R + p.nr - 1) / p.nr);
    const int64_t pairs = K / 128;  // a split holds whole pairs of steps (a stage of MX codes)
    int64_t n = resident / wgs;
    // A split shortens shrink and lengthens expand, which adds them up (rank 128, 1024 rows, K = 13824: 84 us with 6 splits,
    // 170 with 27; rank 32, 4096 rows, K = 5120: 32 with 4, 39 with 10). At few rows shrink takes about 0.57 us more
    // for a pair of steps and expand 1.3 for a split at rank 32, 1.7 and 5 at 128: least where n^2 is 0.34 to 0.44 of the pairs.
    while (n > 1 && 5 * n * n > 2 * pairs) --n;
    if (n < 1) n = 1;
    const int64_t per = (pairs + n - 1) / n;
    p.splits = (int)((pairs + per - 1) / per);
    p.chunks_per_split = (int)(2 * per);
    p.slots = adapters > 1 ? 2 : 1;
    return p;
  }
  const int64_t wgs = (T + kRows - 1) / kRows * ((R + 16 * kRankTiles - 1) / (16 * kRankTiles));
  const int64_t chunks = (K + 127) / 128;
  int64_t n = (512 + wgs - 1) / wgs;
  if (n > (chunks + 3) / 4) n = (chunks + 3) / 4;
  const int64_t per = (chunks + n - 1) / n;
  p.splits = (int)((chunks + per - 1) / per);
  p.chunks_per_split = (int)per;
  // a slot for every adapter that a tile may hold, while that does not make more workgroups than fill the chip
  int64_t slots = T < kRows ? T : kRows;
  if (slots > adapters) slots = adapters;
  if (slots > 1024 / (wgs * p.splits) + 1) slots = 1024 / (wgs * p.splits) + 1;
  p.slots = (int)slots;
  return p;
}

// Lets a kernel have more than 64 KB of LDS, once per device.
template <typename F>
bool lds_limit(F* kernel, int bytes) {
  static int allowed[64] = {0};
  int dev = 0;
  if (bytes <= 60 * 1024) return true;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return false;
  if (dev < 64 && allowed[dev] >= bytes) return true;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  if (dev < 64) allowed[dev] = bytes;
  return true;
}

template <bool kMx, int kNR>
int launch_big(const LoraArgs& a, hipStream_t s) {
  using P = Big<kMx, kNR>;
  WANMI_REQUIRE(lds_limit(&lora_shrink_kernel<kMx, kNR>, P::kLds), WANMI_ERR_HIP, "wanmi_lora_add: %d bytes of LDS refused", P::kLds);
  const dim3 grid((unsigned)((a.T + P::kRows - 1) / P::kRows), (unsigned)((a.R + kNR - 1) / kNR), (unsigned)(a.splits * a.slots));
  hipLaunchKernelGGL((lora_shrink_kernel<kMx, kNR>), grid, dim3(64 * P::kWaves), P::kLds, s, a);
  return check_launch("wanmi_lora_add");
}

// The workgroups of `span` columns that each part takes; their number.
unsigned count_blocks(LoraArgs& a) {
  unsigned blocks = 0;
  for (int i = 0; i < a.parts; ++i) {
    const int w = a.part_end[i] - (i ? a.part_end[i - 1] : 0);
    a.part_blocks[i] = (w + a.span - 1) / a.span;
    blocks += (unsigned)a.part_blocks[i];
  }
  return blocks;
}

template <int kRG, int kKS>
int launch_expand(LoraArgs& a, hipStream_t s) {
  const int ks = kKS > 0 ? kKS : (a.r + 31) / 32;
  const int bytes = kRG * ks * 2048;
  WANMI_REQUIRE(lds_limit(&lora_expand_kernel<kRG, kKS>, bytes), WANMI_ERR_HIP, "wanmi_lora_add: %d bytes of LDS refused", bytes);
  a.span = 256;
  const dim3 grid((unsigned)((a.T + 16 * kRG - 1) / (16 * kRG)), count_blocks(a), (unsigned)a.slots);
  hipLaunchKernelGGL((lora_expand_kernel<kRG, kKS>), grid, dim3(256), bytes, s, a);
  return check_launch("wanmi_lora_add");
}

template <int kKS>
int launch_expand_many(LoraArgs& a, hipStream_t s) {
  using P = Many<kKS>;
  WANMI_REQUIRE(lds_limit(&lora_expand_many_kernel<kKS>, P::kLds), WANMI_ERR_HIP, "wanmi_lora_add: %d bytes of LDS refused", P::kLds);
  // As few workgroups as fill 256 CUs once, three to a CU (ranks up to 64), or twice, two to a CU: a workgroup's start (its
  // ids, its rows' u) costs as much as several blocks of columns, but where requests meet a workgroup takes twice
  // as long, which the second round hides in part. 32768 rows x 5120 columns, one request / three of any
  // length: rank 128 in one round 141 / 210 us, in two 151 / 182; rank 64 in one 132, in two 147.
  const int64_t tiles = (a.T + 127) / 128, resident = kKS == 4 ? 1024 : 768;
  int64_t blocks = (a.N + 63) / 64, each = (blocks * tiles + resident - 1) / resident;
  if (each > blocks) each = blocks;
  a.span = 64 * (int)each;
  const dim3 grid((unsigned)tiles, count_blocks(a));
  hipLaunchKernelGGL((lora_expand_many_kernel<kKS>), grid, dim3(256), P::kLds, s, a);
  return check_launch("wanmi_lora_add");
}

}  // namespace
}  // namespace wanmi

extern "C" int64_t wanmi_lora_workspace(int64_t T, int64_t K, int parts, int rank) {
  using namespace wanmi;
  if (T <= 0 || K <= 0 || parts <= 0 || rank <= 0) return 0;
  const int64_t R = (int64_t)parts * rank;
  // (the splits do not depend on the number of adapters)
  const int n1 = lora_plan(T, K, R, 1, true).splits, n2 = lora_plan(T, K, R, 1, false).splits;
  return (int64_t)sizeof(float) * (n1 > n2 ? n1 : n2) * T * R;
}

extern "C" int wanmi_lora_add(const void* x, const uint8_t* x_scales, const float* row_scale, int64_t ldx, const void* A,
                              const void* B, const float* adapter_scales, const int32_t* adapter_ids,
                              const int32_t* request_ids, int64_t requests, int64_t adapters, int64_t T, int64_t K, int64_t N,
                              int rank, int parts, const int64_t* part_widths, const void* base, int64_t ldb, void* out,
                              int64_t ldo, int zero_rest, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace wanmi;
  clear_error();
  const char* const f = "wanmi_lora_add";
  WANMI_REQUIRE(T >= 0 && T < (1LL << 28), WANMI_ERR_ARG, "%s: T=%lld must be in [0, 2^28)", f, (long long)T);
  WANMI_REQUIRE(K > 0 && K % 32 == 0 && K < (1LL << 24), WANMI_ERR_ARG, "%s: K=%lld must be a positive multiple of 32 below 2^24", f, (long long)K);
  WANMI_REQUIRE(N > 0 && N % 8 == 0 && N < (1LL << 24), WANMI_ERR_ARG, "%s: N=%lld must be a positive multiple of 8 below 2^24", f, (long long)N);
  WANMI_REQUIRE(rank > 0 && rank % 16 == 0 && rank <= 1024, WANMI_ERR_ARG, "%s: rank=%d must be a multiple of 16, at most 1024 (pad with zeros)", f, rank);
  WANMI_REQUIRE(parts >= 1 && parts <= kMaxParts && part_widths, WANMI_ERR_ARG, "%s: parts=%d must be 1 to %d", f, parts, kMaxParts);
  WANMI_REQUIRE(adapters >= 1 && adapters < (1LL << 24), WANMI_ERR_ARG, "%s: adapters=%lld must be 1 to 2^24", f, (long long)adapters);
  WANMI_REQUIRE(requests >= 0 && requests < (1LL << 31), WANMI_ERR_ARG, "%s: requests=%lld out of range", f, (long long)requests);
  LoraArgs a;
  int64_t end = 0;
  for (int i = 0; i < parts; ++i) {
    WANMI_REQUIRE(part_widths[i] > 0 && part_widths[i] <= N - end && (parts == 1 || part_widths[i] % 64 == 0), WANMI_ERR_ARG,
                  "%s: part %d is %lld columns wide: multiples of 64 that sum to N", f, i, (long long)part_widths[i]);
    end += part_widths[i];
    a.part_end[i] = (int)end;
  }
  WANMI_REQUIRE(end == N, WANMI_ERR_ARG, "%s: the parts hold %lld of %lld columns", f, (long long)end, (long long)N);
  if (T == 0) return WANMI_OK;
  // (without requests there is no row that has an adapter id)
  WANMI_REQUIRE(x && A && B && (adapter_ids || (request_ids && requests == 0)) && base && out && workspace, WANMI_ERR_ARG, "%s: null pointer", f);
  WANMI_REQUIRE(ldx >= K && ldx % (x_scales ? 16 : 8) == 0, WANMI_ERR_ARG, "%s: x rows must be 16-byte aligned", f);
  WANMI_REQUIRE(ldb >= N && ldb % 8 == 0 && ldo >= N && ldo % 8 == 0, WANMI_ERR_ARG,
                "%s: the row strides of base and out must be multiples of 8 of at least N", f);
  for (const void* p : {x, A, B, base, (const void*)out, (const void*)workspace})
    WANMI_REQUIRE(((uintptr_t)p % 16) == 0, WANMI_ERR_ARG, "%s: tensors must be 16-byte aligned", f);
  const int64_t need = wanmi_lora_workspace(T, K, parts, rank);
  WANMI_REQUIRE(workspace_bytes >= need, WANMI_ERR_ARG, "%s: the workspace holds %lld bytes, %lld are needed", f,
                (long long)workspace_bytes, (long long)need);
  a.x = x;
  a.x_scales = x_scales;
  a.row_scale = row_scale;
  a.ldx = ldx;
  a.ldxs = K / 32;
  a.A = static_cast<const uint16_t*>(A);
  a.B = static_cast<const uint16_t*>(B);
  a.scales = adapter_scales;
  a.adapter_ids = adapter_ids;
  a.request_ids = request_ids;
  a.requests = (int)requests;
  a.adapters = (int)adapters;
  a.T = T;
  a.K = (int)K;
  a.N = (int)N;
  a.r = rank;
  a.R = parts * rank;
  a.parts = parts;
  const LoraPlan plan = lora_plan(T, K, a.R, adapters, ldx < (1LL << 21) && (uintptr_t)x_scales % 4 == 0);
  a.splits = plan.splits;
  a.chunks_per_split = plan.chunks_per_split;
  a.slots = plan.slots;
  a.in_place = base == out && ldb == ldo;
  a.u = static_cast<float*>(workspace);
  a.base = static_cast<const uint16_t*>(base);
  a.ldb = ldb;
  a.out = static_cast<uint16_t*>(out);
  a.ldo = ldo;
  a.zero_rest = zero_rest;
  hipStream_t s = (hipStream_t)stream;
  int st;
  if (plan.big) {
    if (x_scales) st = plan.nr == 32 ? launch_big<true, 32>(a, s) : plan.nr == 64 ? launch_big<true, 64>(a, s) : launch_big<true, 128>(a, s);
    else st = plan.nr == 32 ? launch_big<false, 32>(a, s) : plan.nr == 64 ? launch_big<false, 64>(a, s) : launch_big<false, 128>(a, s);
  } else {
    const dim3 grid((unsigned)((T + kRows - 1) / kRows), (unsigned)((a.R + 16 * kRankTiles - 1) / (16 * kRankTiles)), (unsigned)(a.splits * a.slots));
    if (x_scales) hipLaunchKernelGGL((lora_shrink_few_kernel<true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((lora_shrink_few_kernel<false>), grid, dim3(256), 0, s, a);
    st = check_launch(f);
  }
  if (st != WANMI_OK) return st;
  if (T >= 1024 && rank <= 128 && ldb < (1 << 22) && ldo < (1 << 22) && N * rank < (1LL << 30))
    return rank <= 32 ? launch_expand_many<1>(a, s) : rank <= 64 ? launch_expand_many<2>(a, s) : launch_expand_many<4>(a, s);
  return rank <= 32 ? launch_expand<2, 1>(a, s) : rank <= 64 ? launch_expand<2, 2>(a, s) : launch_expand<2, 0>(a, s);
}
