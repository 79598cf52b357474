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
// second product takes it as the sum of two bf16 values (u to 2^-17): an error of 2^-9 per rank would be
// as large as the output's own rounding where the adapter outweighs the base.
//
// The MFMA's rows are ranks (shrink) and output columns (expand), its columns tokens, so that a lane ends with
// consecutive ranks or columns of one token. The order of k inside a product is free as long as both
// operands agree: a lane takes 32 consecutive k (one MX block: one scale) for the four MFMAs of a chunk of 128.
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
  int splits, chunks_per_split;
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
  int64_t at = t;
  if (a.request_ids) {
    const int q = a.request_ids[t];
    if ((uint32_t)q >= (uint32_t)a.requests) return -2;
    at = q;
  }
  const int e = a.adapter_ids[at];
  return (uint32_t)e < (uint32_t)a.adapters ? e : -1;
}

constexpr int kRows = 32;  // rows of a tile: two MFMA columns
constexpr int kRankTiles = 4;

template <bool kMx>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraArgs a) {
  __shared__ f32x4 red[4][2 * kRankTiles][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t t0 = (int64_t)blockIdx.x * kRows;
  const int rank0 = blockIdx.y * 16 * kRankTiles;
  const int split = blockIdx.z;
  const int nchunks = (a.K + 127) / 128;
  const int ch0 = split * a.chunks_per_split, ch1 = min(ch0 + a.chunks_per_split, nchunks);
  const int mine = lane < kRows ? row_adapter(a, t0 + lane) : -2;
  uint64_t todo = __ballot(mine >= 0);
  int64_t row[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) row[m] = min(t0 + 16 * m + c, a.T - 1);  // rows past the end: loaded again, not used
  while (todo) {
    const int e = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    const uint64_t match = __ballot(mine == e);
    todo &= ~match;
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
          for (int s = 0; s < 4; ++s) {
            union { bf16x8 v; bf16x2_t p[4]; } f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t d = w[s >> 1][2 * (s & 1) + j];
              f.p[2 * j] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, sc, false);
              f.p[2 * j + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d, sc, true);
            }
            xf[m][s] = f.v;
          }
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

// A wave: kRows rows x 64 columns. Row i of MFMA operand tile s stands for column n0 + 16 (i / 4) + 4 s + i % 4, so that
// over the four tiles a lane holds 16 consecutive columns of its token.
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int64_t t0 = (int64_t)blockIdx.x * kRows;
  const int n0 = (blockIdx.y * 4 + wave) * 64;
  if (n0 >= a.N) return;
  const int mine = lane < kRows ? row_adapter(a, t0 + lane) : -2;
  uint64_t todo = __ballot(mine >= 0);
  int part = 0;
  while (part < a.parts - 1 && n0 >= a.part_end[part]) ++part;
  f32x4 acc[2][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int s = 0; s < 4; ++s) acc[m][s] = f32x4{0.f, 0.f, 0.f, 0.f};
  while (todo) {
    const int e = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    const uint64_t match = __ballot(mine == e);
    todo &= ~match;
    f32x4 tmp[2][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < 4; ++s) tmp[m][s] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < a.r; k0 += 32) {
      const int k = k0 + 8 * g;
      bf16x8 bf[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int n = min(n0 + 16 * (c >> 2) + 4 * s + (c & 3), a.N - 1);
        u32x4 v = {0u, 0u, 0u, 0u};
        if (k < a.r) v = *reinterpret_cast<const u32x4*>(a.B + ((int64_t)e * a.N + n) * a.r + k);
        bf[s] = __builtin_bit_cast(bf16x8, v);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.0f;
        if (k < a.r && (match >> (16 * m + c) & 1)) {
          const float* pu = a.u + (t0 + 16 * m + c) * a.R + part * a.r + k;
          for (int q = 0; q < a.splits; ++q, pu += a.T * a.R) {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(pu), hi = *reinterpret_cast<const f32x4*>(pu + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] += lo[j], f[4 + j] += hi[j];
          }
        }
        // u = uh + ul, two bf16 values; an infinity is uh alone
        u32x4 uh, ul;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uh[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
          const float h0 = bf16_lo(uh[j]), h1 = bf16_hi(uh[j]);
          ul[j] = pack_bf16x2(fabsf(h0) < INFINITY ? f[2 * j] - h0 : 0.0f, fabsf(h1) < INFINITY ? f[2 * j + 1] - h1 : 0.0f);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          tmp[m][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[s], __builtin_bit_cast(bf16x8, uh), tmp[m][s], 0, 0, 0);
          tmp[m][s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[s], __builtin_bit_cast(bf16x8, ul), tmp[m][s], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (match >> (16 * m + c) & 1) acc[m][s] = tmp[m][s];
  }
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int64_t t = t0 + 16 * m + c;
    const int e = __shfl(mine, 16 * m + c, 64);
    if (t >= a.T || (e == -2 && !a.zero_rest)) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n0 + 16 * g + 8 * h;
      if (n + 8 > a.N) continue;
      u32x4 o = {0u, 0u, 0u, 0u};
      if (e != -2) {
        o = *reinterpret_cast<const u32x4*>(a.base + t * a.ldb + n);
        if (e >= 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = pack_bf16x2(bf16_lo(o[j]) + acc[m][2 * h + j / 2][2 * (j & 1)],
                               bf16_hi(o[j]) + acc[m][2 * h + j / 2][2 * (j & 1) + 1]);
        }
      }
      store_b128_guarded(o, a.out + t * a.ldo + n);
    }
  }
}

int splits_for(int64_t T, int64_t K, int64_t R) {
  const int64_t tiles = (T + kRows - 1) / kRows * ((R + 16 * kRankTiles - 1) / (16 * kRankTiles));
  const int64_t chunks = (K + 127) / 128;
  int64_t n = (512 + tiles - 1) / tiles;
  const int64_t most = (chunks + 3) / 4;
  if (n > most) n = most;
  const int64_t per = (chunks + n - 1) / n;
  return (int)((chunks + per - 1) / per);
}

}  // namespace
}  // namespace wanmi

extern "C" int64_t wanmi_lora_workspace(int64_t T, int64_t K, int parts, int rank) {
  using namespace wanmi;
  if (T <= 0 || K <= 0 || parts <= 0 || rank <= 0) return 0;
  return (int64_t)sizeof(float) * splits_for(T, K, (int64_t)parts * rank) * T * parts * rank;
}

extern "C" int wanmi_lora_add(const void* x, const uint8_t* x_scales, const float* row_scale, int64_t ldx, const void* A,
                              const void* B, const float* adapter_scales, const int32_t* adapter_ids,
                              const int32_t* request_ids, int64_t requests, int64_t adapters, int64_t T, int64_t K, int64_t N,
                              int rank, int parts, const int64_t* part_widths, const void* base, int64_t ldb, void* out,
                              int64_t ldo, int zero_rest, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace wanmi;
  clear_error();
  const char* const f = "wanmi_lora_add";
  WANMI_REQUIRE(T >= 0 && T < (1LL << 31), WANMI_ERR_ARG, "%s: T=%lld must be in [0, 2^31)", f, (long long)T);
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
  WANMI_REQUIRE(x && A && B && adapter_ids && base && out && workspace, WANMI_ERR_ARG, "%s: null pointer", f);
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
  a.splits = splits_for(T, K, a.R);
  const int chunks = (int)((K + 127) / 128);
  a.chunks_per_split = (chunks + a.splits - 1) / a.splits;
  a.u = static_cast<float*>(workspace);
  a.base = static_cast<const uint16_t*>(base);
  a.ldb = ldb;
  a.out = static_cast<uint16_t*>(out);
  a.ldo = ldo;
  a.zero_rest = zero_rest;
  hipStream_t s = (hipStream_t)stream;
  const unsigned tiles = (unsigned)((T + kRows - 1) / kRows);
  const dim3 g1(tiles, (unsigned)((a.R + 16 * kRankTiles - 1) / (16 * kRankTiles)), (unsigned)a.splits);
  if (x_scales) hipLaunchKernelGGL((lora_shrink_kernel<true>), g1, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((lora_shrink_kernel<false>), g1, dim3(256), 0, s, a);
  const int st = check_launch(f);
  if (st != WANMI_OK) return st;
  hipLaunchKernelGGL(lora_expand_kernel, dim3(tiles, (unsigned)((N + 255) / 256)), dim3(256), 0, s, a);
  return check_launch(f);
}
