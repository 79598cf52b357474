// Norms before and after a sub-layer, fused with its gate and residual scale, for packed batches (gfx950).
//
//   p = Norm_post(hidden) * post_weight                        (fp32)
//   r = bf16(alpha * residual + gate[q] * p)                   the carried residual, written (residual optional)
//   y = bf16(Norm_pre(r) * mul[q] + add[q])                    written as it is, as MX or as ROW codes, or not wanted
//
// for every row of a packed [T, H] batch, q the row's request: gate, mul and add are one row of H
// for all requests or one per request. A row whose id names no request is not computed: it is left as it
// was, or written as zeros where the caller has just allocated the outputs.
//
// The sum r is the only value between the input and y that is rounded (it is an output, and the norm that
// follows in the block reads it again). Statistics are fp32: each wave takes the mean of its own columns, then the sum
// of squared deviations from that, and the waves' means and sums are joined exactly (no difference of large
// sums is taken).
//
// The vectors are 16 bytes a column against the row's own 8, so where they are read from decides the pass: from L2 for every
// row, 32760 rows of 5120 took 349 us. Two kernels:
//
// Many rows: a wavefront owns a row, lane l the columns 512 c + 8 l .. + 7 of every chunk c; a workgroup of eight copies the
// vectors of its rows' request into LDS while the rows are under way (where the eight rows belong to several requests, each
// wave reads its own from L2). A wave takes one row and ends: in a loop, the loads of the next row stand
// behind the stores of this one in the order that a wave waits for them, and 32760 rows took 343 us instead of 257
// (5.2 TB/s of the 5.5 that a large copy reaches here; with MX codes 226 to 231, ROW 237 to 247, without and with a norm
// before the gate).
//
// Few rows: a workgroup owns a row, a thread 8 columns of it (kNC runs of them), so that all of its waves share the
// row's latency: 5.5 us for 7 rows where a wavefront each takes 12.
#include <type_traits>

#include "wanmi_common.h"

namespace wanmi {

struct SandwichArgs {
  const uint16_t* hidden;
  const uint16_t* residual;
  int64_t ld_h, ld_r;
  const float* post_weight;
  const float* gate;
  const float* mul;
  const float* add;
  int64_t ld_gate, ld_mul, ld_add;  // elements between requests; 0: one row for every request
  const int32_t* ids;
  int requests;
  float alpha, eps;
  int64_t T, rows_each;  // rows of a workgroup
  int H;
  int post_norm, norm, quant;
  int zero_rest;
  uint16_t* residual_out;
  void* out;
  uint8_t* scales;
};

namespace {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kMaxWaves = 16;
constexpr int kRsrcWord3 = 0x00020000;  // gfx9 raw buffer descriptor word 3

// A buffer descriptor over `bytes` bytes at `p`; accesses past the end read 0 / are dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, kRsrcWord3);
}

// MX codes of the lane's 8 columns of a block of 32 (4 consecutive lanes), and the block's biased exponent: that of its
// largest |y|, less 7.
__device__ __forceinline__ int mx_codes(const uint32_t (&y)[4], u32x2& codes) {
  u16x2 mag = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) mag = __builtin_elementwise_max(mag, __builtin_bit_cast(u16x2, y[j] & 0x7FFF7FFFu));
  int e = (int)(max(mag[0], mag[1]) >> 7);
  e = max(e, dpp_i32<0xB1>(e));
  e = max(e, dpp_i32<0x4E>(e));
  const int sexp = max(e - 7, 0);
  const float f = mx_inv_scale(sexp);
  codes[0] = cvt_e4m3x4(bf16_lo(y[0]) * f, bf16_hi(y[0]) * f, bf16_lo(y[1]) * f, bf16_hi(y[1]) * f);
  codes[1] = cvt_e4m3x4(bf16_lo(y[2]) * f, bf16_hi(y[2]) * f, bf16_lo(y[3]) * f, bf16_hi(y[3]) * f);
  return sexp;
}

// ROW codes of 8 columns: e4m3(y / dq), clamped to the largest code.
__device__ __forceinline__ u32x2 row_codes(const uint32_t (&y)[4], float dq) {
  float q[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    q[2 * j] = fminf(fmaxf(bf16_lo(y[j]) / dq, -448.0f), 448.0f);
    q[2 * j + 1] = fminf(fmaxf(bf16_hi(y[j]) / dq, -448.0f), 448.0f);
  }
  return u32x2{cvt_e4m3x4(q[0], q[1], q[2], q[3]), cvt_e4m3x4(q[4], q[5], q[6], q[7])};
}

// 8 consecutive floats of a vector into registers; `none` where there is no vector or no column.
__device__ __forceinline__ void load8(const float* p, int col, bool ok, float none, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = none;
  if (p && ok) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p + col), hi = *reinterpret_cast<const f32x4*>(p + col + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = lo[j], v[4 + j] = hi[j];
  }
}

__device__ __forceinline__ float sum8(const float (&v)[8]) {
  return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// How many of the row's columns wave w of the workgroup holds.
template <int kNC>
__device__ __forceinline__ float columns_of(int w, int waves, int H) {
  int n = 0;
#pragma unroll
  for (int c = 0; c < kNC; ++c) n += max(0, min(512, H - (c * waves + w) * 512));
  return w < waves ? (float)n : 0.0f;
}

// Mean and 1 / sqrt(variance, or mean square, + eps) of the row whose columns the workgroup's threads hold as x (fp32;
// zero past H). `part` [waves][2] in LDS: this reduction's own; one barrier. mine, theirs: columns of this wave and of
// wave number `lane`, which is the one whose part a lane takes into the joined sums.
template <int kNC>
__device__ __forceinline__ void row_stats(const float (&x)[kNC][8], const bool (&ok)[kNC], int norm, float H, float eps, int wave,
                                          float mine, float theirs, float (*part)[2], float& mu, float& rs) {
  mu = 0.0f;
  rs = 1.0f;
  if (norm == WANMI_NORM_NONE) return;
  const int lane = threadIdx.x & 63;
  float mw = 0.0f;  // the mean of the wave's columns
  if (norm == WANMI_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < kNC; ++c) s += sum8(x[c]);
    mw = mine > 0.0f ? wave_sum_f32_asc(s) / mine : 0.0f;
  }
  float q = 0.0f;
#pragma unroll
  for (int c = 0; c < kNC; ++c) {
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = (x[c][j] - mw) * (x[c][j] - mw);
    q += ok[c] ? sum8(d) : 0.0f;
  }
  q = wave_sum_f32_asc(q);
  if (lane == 0) {
    part[wave][0] = mw;
    part[wave][1] = q;
  }
  __syncthreads();
  float m = part[lane & (kMaxWaves - 1)][0], t = part[lane & (kMaxWaves - 1)][1];
  t = theirs > 0.0f ? t : 0.0f;
  if (norm == WANMI_NORM_LAYER) {
    m = theirs > 0.0f ? m : 0.0f;
    mu = wave_sum_f32_asc(theirs * m) / H;
    t += theirs * (m - mu) * (m - mu);
  }
  rs = rsqrt_f32(wave_sum_f32_asc(t) / H + eps);
}

template <int kNC>
__global__ __launch_bounds__(64 * kMaxWaves) __attribute__((amdgpu_waves_per_eu(kNC == 1 ? 5 : 4))) void adaln_sandwich_few_kernel(SandwichArgs a) {
  __shared__ float part[2][2][kMaxWaves][2];  // [row parity][norm][wave]
  __shared__ float top[2][kMaxWaves];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
  const int H = a.H;
  const int64_t row0 = (int64_t)blockIdx.x * a.rows_each, row1 = min(row0 + a.rows_each, a.T);
  int col[kNC];
  bool ok[kNC];
#pragma unroll
  for (int c = 0; c < kNC; ++c) {
    col[c] = 8 * (tid + c * (int)blockDim.x);
    ok[c] = col[c] < H;
  }
  const float mine = columns_of<kNC>(wave, waves, H), theirs = columns_of<kNC>(tid & 63, waves, H);
  const u32x4 zero = {0u, 0u, 0u, 0u};
  const int64_t out_bytes = a.quant == WANMI_QUANT_NONE ? 2 * (int64_t)H : a.quant == WANMI_QUANT_MX ? (int64_t)H : (int64_t)H + 4;

  float wv[kNC][8], gv[kNC][8], mv[kNC][8], av[kNC][8];
#pragma unroll
  for (int c = 0; c < kNC; ++c) load8(a.post_weight, col[c], ok[c], 1.0f, wv[c]);
  int held = -1;  // the request whose vectors are in registers

  u32x4 hn[kNC], rn[kNC];
  const auto fetch = [&](int64_t row) {
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
      hn[c] = ok[c] ? *reinterpret_cast<const u32x4*>(a.hidden + row * a.ld_h + col[c]) : zero;
      rn[c] = ok[c] && a.residual ? *reinterpret_cast<const u32x4*>(a.residual + row * a.ld_r + col[c]) : zero;
    }
  };
  // the requests of the rows, 64 at a time (one a lane), so that a row's fetch does not wait for its id
  int ids = 0;
  const auto request = [&](int64_t row) {
    const int k = (int)(row - row0) & 63;
    if (k == 0 && a.ids) ids = a.ids[min(row + (tid & 63), a.T - 1)];
    return __builtin_amdgcn_readlane(ids, k);
  };
  int id = request(row0), par = 0;  // par: of the rows computed, so that no row writes the sums that the one before it reads
  if ((uint32_t)id < (uint32_t)a.requests) fetch(row0);
  for (int64_t row = row0; row < row1; ++row) {
    const bool live = (uint32_t)id < (uint32_t)a.requests;
    const int next = row + 1 < row1 ? request(row + 1) : -1;
    uint16_t* ro = a.residual_out + row * H;
    uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + row * out_bytes;
    if (!live) {
      if (a.zero_rest) {
#pragma unroll
        for (int c = 0; c < kNC; ++c) {
          if (!ok[c]) continue;
          store_b128_guarded(zero, ro + col[c]);
          if (!a.out) {
          } else if (a.quant == WANMI_QUANT_NONE) {
            store_b128_guarded(zero, out + 2 * col[c]);
          } else if (a.quant == WANMI_QUANT_MX) {
            *reinterpret_cast<u32x2*>(out + col[c]) = u32x2{0u, 0u};
            if ((tid & 3) == 0) a.scales[row * (int64_t)(H / 32) + col[c] / 32] = 0;
          } else {  // (rows of H + 4 bytes: 4-byte aligned)
            reinterpret_cast<uint32_t*>(out + col[c])[0] = 0u;
            reinterpret_cast<uint32_t*>(out + col[c])[1] = 0u;
          }
        }
        if (a.out && a.quant == WANMI_QUANT_ROW && tid == 0) *reinterpret_cast<uint32_t*>(out + H) = 0u;
      }
      id = next;
      if ((uint32_t)id < (uint32_t)a.requests) fetch(row + 1);
      continue;  // (id is the same for the whole workgroup)
    }
    if (id != held) {
      held = id;
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
        load8(a.gate ? a.gate + id * a.ld_gate : nullptr, col[c], ok[c], 1.0f, gv[c]);
        load8(a.mul ? a.mul + id * a.ld_mul : nullptr, col[c], ok[c], 1.0f, mv[c]);
        load8(a.add ? a.add + id * a.ld_add : nullptr, col[c], ok[c], 0.0f, av[c]);
      }
    }
    float x[kNC][8];
    u32x4 r[kNC];
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[c][2 * j] = bf16_lo(hn[c][j]), x[c][2 * j + 1] = bf16_hi(hn[c][j]);
      r[c] = rn[c];
    }
    if ((uint32_t)next < (uint32_t)a.requests) fetch(row + 1);
    float mu, rs;
    row_stats<kNC>(x, ok, a.post_norm, (float)H, a.eps, wave, mine, theirs, part[par][0], mu, rs);
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p0 = (x[c][2 * j] - mu) * rs * wv[c][2 * j], p1 = (x[c][2 * j + 1] - mu) * rs * wv[c][2 * j + 1];
        r[c][j] = pack_bf16x2(a.alpha * bf16_lo(r[c][j]) + gv[c][2 * j] * p0, a.alpha * bf16_hi(r[c][j]) + gv[c][2 * j + 1] * p1);
        x[c][2 * j] = ok[c] ? bf16_lo(r[c][j]) : 0.0f;
        x[c][2 * j + 1] = ok[c] ? bf16_hi(r[c][j]) : 0.0f;
      }
      if (ok[c]) store_b128_guarded(r[c], ro + col[c]);
    }
    if (!a.out) {  // (the same for the whole workgroup)
      id = next;
      par ^= 1;
      continue;
    }
    row_stats<kNC>(x, ok, a.norm, (float)H, a.eps, wave, mine, theirs, part[par][1], mu, rs);
    float amax = 0.0f;
    uint32_t y[kNC][4];
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y0 = (x[c][2 * j] - mu) * rs * mv[c][2 * j] + av[c][2 * j];
        const float y1 = (x[c][2 * j + 1] - mu) * rs * mv[c][2 * j + 1] + av[c][2 * j + 1];
        y[c][j] = ok[c] ? pack_bf16x2(y0, y1) : 0u;
      }
      if (a.quant == WANMI_QUANT_NONE) {
        if (ok[c]) store_b128_guarded(u32x4{y[c][0], y[c][1], y[c][2], y[c][3]}, out + 2 * col[c]);
      } else if (a.quant == WANMI_QUANT_MX) {
        u32x2 cv;
        const int sexp = mx_codes(y[c], cv);
        if (ok[c]) {
          *reinterpret_cast<u32x2*>(out + col[c]) = cv;
          if ((tid & 3) == 0) a.scales[row * (int64_t)(H / 32) + col[c] / 32] = (uint8_t)sexp;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(y[c][j])), fabsf(bf16_hi(y[c][j]))));
      }
    }
    if (a.quant == WANMI_QUANT_ROW) {
      amax = wave_max_f32_asc(amax);
      if ((tid & 63) == 0) top[par][wave] = amax;
      __syncthreads();
      for (int w = 0; w < waves; ++w) amax = fmaxf(amax, top[par][w]);
      const float dq = fmaxf(amax / 448.0f, 1e-6f);
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
        if (!ok[c]) continue;
        const u32x2 cv = row_codes(y[c], dq);  // (rows of H + 4 bytes: 4-byte aligned)
        reinterpret_cast<uint32_t*>(out + col[c])[0] = cv[0];
        reinterpret_cast<uint32_t*>(out + col[c])[1] = cv[1];
      }
      if (tid == 0) *reinterpret_cast<float*>(out + H) = dq;
    }
    id = next;
    par ^= 1;
  }
}

// ------------------------------------------------------------------------------------------------
// Many rows
// ------------------------------------------------------------------------------------------------
// Mean and 1 / sqrt(variance, or mean square, + eps) of a row held by one wave, columns as `at(c, j)` gives them; those
// past H (in the last chunk alone: `inside`) are zero.
template <int NCH, typename F, typename G>
__device__ __forceinline__ void wave_stats(const F& at, const G& packed, int norm, bool inside, float H, float eps, float& mu, float& rs) {
  mu = 0.0f;
  rs = 1.0f;
  if (norm == WANMI_NORM_NONE) return;
  float q = 0.0f;
  if (norm == WANMI_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      s += ((at(c, 0) + at(c, 1)) + (at(c, 2) + at(c, 3))) + ((at(c, 4) + at(c, 5)) + (at(c, 6) + at(c, 7)));
    mu = wave_sum_f32_asc(s) / H;
    packed();
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      float d[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = at(c, j) - mu;
      const float t = ((d[0] * d[0] + d[1] * d[1]) + (d[2] * d[2] + d[3] * d[3])) + ((d[4] * d[4] + d[5] * d[5]) + (d[6] * d[6] + d[7] * d[7]));
      q += c < NCH - 1 || inside ? t : 0.0f;
    }
  } else {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      float d[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = at(c, j);
      q += ((d[0] * d[0] + d[1] * d[1]) + (d[2] * d[2] + d[3] * d[3])) + ((d[4] * d[4] + d[5] * d[5]) + (d[6] * d[6] + d[7] * d[7]));
    }
  }
  rs = rsqrt_f32(wave_sum_f32_asc(q) / H + eps);
  packed();
}

// The four vectors in LDS: vector v, chunk c as lane-major 16-byte pieces, every lane's first four floats, then every
// lane's second four, so that a lane's reads of a chunk are consecutive across lanes.
// NCH is the row's number of chunks exactly: no chunk is conditional, and the loads, LDS reads and arithmetic of
// several overlap.
constexpr int kManyWaves = 8;

template <int NCH>
__global__ __launch_bounds__(64 * kManyWaves) __attribute__((amdgpu_waves_per_eu(4))) void adaln_sandwich_kernel(SandwichArgs a) {
  extern __shared__ __attribute__((aligned(1024))) float vecs[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int nch = NCH, waves = kManyWaves;
  const int H = a.H;
  const bool inside = (NCH - 1) * 512 + lane * 8 < H;  // the lane's columns of the last chunk
  const int64_t row0 = (int64_t)blockIdx.x * waves;
  const int64_t out_bytes = a.quant == WANMI_QUANT_NONE ? 2 * (int64_t)H : a.quant == WANMI_QUANT_MX ? (int64_t)H : (int64_t)H + 4;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  const uint32_t base = lds_addr(vecs);
  int held = -1;  // the request whose vectors lie in LDS
  const auto vector = [&](int v, int id) -> const float* {
    return v == 0 ? a.post_weight
           : v == 1 ? (a.gate ? a.gate + id * a.ld_gate : nullptr)
           : v == 2 ? (a.mul ? a.mul + id * a.ld_mul : nullptr)
                    : (a.add ? a.add + id * a.ld_add : nullptr);
  };

  const int64_t row = row0 + wave, from = min(row, a.T - 1);
  // the row is under way while its request is looked up and the vectors are copied
  constexpr int kAhead = NCH <= 6 ? NCH : 4;  // chunks of the residual under way (all of it where the registers hold it)
  uint32_t xp[NCH][4], rp[kAhead][4];
  const __amdgpu_buffer_rsrc_t r_x = rsrc(a.hidden + from * a.ld_h, 2 * (int64_t)H);
  const __amdgpu_buffer_rsrc_t r_r = rsrc(a.residual ? a.residual + from * a.ld_r : a.hidden + from * a.ld_h, 2 * (int64_t)H);
  // columns past H in the last chunk lie past the descriptors' extents and read as zero
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r_x, lane * 16, c * 1024, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) xp[c][j] = v[j];
  }
#pragma unroll
  for (int c = 0; c < kAhead; ++c) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r_r, lane * 16, c * 1024, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) rp[c][j] = v[j];
  }
  // the workgroup's requests (one a lane); every wave comes to the same decision
  const bool in = lane < waves && row0 + lane < a.T;
  const int theirs = !in ? -1 : a.ids ? a.ids[row0 + lane] : 0;
  const uint64_t alive = __ballot((uint32_t)theirs < (uint32_t)a.requests);
  const int first = alive ? __builtin_amdgcn_readlane(theirs, __builtin_ctzll(alive)) : -1;
  const bool one = alive && __ballot(theirs == first) == alive;
  const int id = __builtin_amdgcn_readlane(theirs, wave);
  const bool live = (uint32_t)id < (uint32_t)a.requests;
  if (one) {
    held = first;
    for (int k = wave; k < 8 * nch; k += waves) {  // 1 KiB pieces: vector, half, chunk
      const int v = k / (2 * nch), half = k / nch % 2, c = k % nch;
      const float* p = vector(v, held);
      const uint32_t to = (uint32_t)((v * 2 + half) * nch + c) * 1024;
      const float none = v == 3 ? 0.0f : 1.0f;
      if (p) lds_dma_b128(buffer_rsrc(p, 4u * (uint32_t)H), (uint32_t)(c * 512 + 8 * lane + 4 * half) * 4, base + to);
      else reinterpret_cast<f32x4*>(vecs)[to / 16 + lane] = f32x4{none, none, none, none};
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    __syncthreads();
  }
  if (row >= a.T) return;
  uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + row * out_bytes;
  const __amdgpu_buffer_rsrc_t r_ro = rsrc(a.residual_out + row * H, 2 * (int64_t)H);
  const __amdgpu_buffer_rsrc_t r_o = rsrc(out, a.quant == WANMI_QUANT_ROW ? (int64_t)H : out_bytes);
  const __amdgpu_buffer_rsrc_t r_s = rsrc(a.quant == WANMI_QUANT_MX && a.out ? a.scales + row * (int64_t)(H / 32) : nullptr,
                                          a.quant == WANMI_QUANT_MX ? H / 32 : 0);
  if (!live) {
    if (!a.zero_rest) return;
    for (int c = 0; c < nch; ++c) {
      store_b128_guarded(zero, r_ro, lane * 16, c * 1024);
      if (!a.out) {
      } else if (a.quant == WANMI_QUANT_NONE) {
        store_b128_guarded(zero, r_o, lane * 16, c * 1024);
      } else {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{0u, 0u}, r_o, lane * 8, c * 512, 0);
        if (a.quant == WANMI_QUANT_MX)
          __builtin_amdgcn_raw_buffer_store_b8((uint8_t)0, r_s, (lane & 3) == 0 ? c * 16 + (lane >> 2) : H, 0, 0);
      }
    }
    if (a.out && a.quant == WANMI_QUANT_ROW && lane == 0) *reinterpret_cast<uint32_t*>(out + H) = 0u;
    return;
  }
  // (the whole row in one piece of straight code for either place of the vectors)
  const auto body = [&](auto where) {
    const auto load = [&](int v, int c, float (&x)[8]) {
      if constexpr (decltype(where)::value) {
        const f32x4 lo = reinterpret_cast<const f32x4*>(vecs)[((v * 2) * nch + c) * 64 + lane];
        const f32x4 hi = reinterpret_cast<const f32x4*>(vecs)[((v * 2 + 1) * nch + c) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = lo[j], x[4 + j] = hi[j];
      } else {
        const int col = c * 512 + lane * 8;
        load8(vector(v, id), col, col < H, v == 3 ? 0.0f : 1.0f, x);
      }
    };

    const auto x = [&](int c, int j) { return (j & 1) ? bf16_hi(xp[c][j >> 1]) : bf16_lo(xp[c][j >> 1]); };
    // between the phases the row is unpacked anew instead of being held as fp32 (which spilled)
    const auto packed = [&]() {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(xp[c][j]));
    };
    float mu, rs;
    wave_stats<NCH>(x, packed, a.post_norm, inside, (float)H, a.eps, mu, rs);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      float wv[8], gv[8];
      load(0, c, wv);
      load(1, c, gv);
      u32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p0 = (bf16_lo(xp[c][j]) - mu) * rs * wv[2 * j], p1 = (bf16_hi(xp[c][j]) - mu) * rs * wv[2 * j + 1];
        o[j] = pack_bf16x2((a.residual ? a.alpha * bf16_lo(rp[c % kAhead][j]) : 0.0f) + gv[2 * j] * p0,
                             (a.residual ? a.alpha * bf16_hi(rp[c % kAhead][j]) : 0.0f) + gv[2 * j + 1] * p1);
        if (c == NCH - 1 && !inside) o[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) xp[c][j] = o[j];
      if (c + kAhead < NCH) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r_r, lane * 16, (c + kAhead) * 1024, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) rp[c % kAhead][j] = v[j];
      }
      store_b128_guarded(o, r_ro, lane * 16, c * 1024);
    }
    if (!a.out) return;
    wave_stats<NCH>(x, packed, a.norm, inside, (float)H, a.eps, mu, rs);
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const bool ok = c < NCH - 1 || inside;
      float mv[8], av[8];
      load(2, c, mv);
      load(3, c, av);
      uint32_t y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y0 = (x(c, 2 * j) - mu) * rs * mv[2 * j] + av[2 * j];
        const float y1 = (x(c, 2 * j + 1) - mu) * rs * mv[2 * j + 1] + av[2 * j + 1];
        y[j] = ok ? pack_bf16x2(y0, y1) : 0u;
      }
      if (a.quant == WANMI_QUANT_NONE) {
        store_b128_guarded(u32x4{y[0], y[1], y[2], y[3]}, r_o, lane * 16, c * 1024);
      } else if (a.quant == WANMI_QUANT_MX) {
        u32x2 cv;
        const int sexp = mx_codes(y, cv);
        __builtin_amdgcn_raw_buffer_store_b64(cv, r_o, lane * 8, c * 512, 0);
        // one byte per 4 lanes; the other lanes' offsets lie past the extent and are dropped
        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)sexp, r_s, ok && (lane & 3) == 0 ? c * 16 + (lane >> 2) : H, 0, 0);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(y[j])), fabsf(bf16_hi(y[j]))));
          xp[c][j] = y[j];
        }
      }
    }
    if (a.quant == WANMI_QUANT_ROW) {
      amax = wave_max_f32_asc(amax);
      const float dq = fmaxf(amax / 448.0f, 1e-6f);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        __builtin_amdgcn_raw_buffer_store_b64(row_codes(xp[c], dq), r_o, lane * 8, c * 512, 0);
      }
      if (lane == 0) *reinterpret_cast<float*>(out + H) = dq;
    }
  };
  if (id == held) body(std::integral_constant<bool, true>{});
  else body(std::integral_constant<bool, false>{});
}

template <int kNC>
void launch_few(const SandwichArgs& a, hipStream_t s) {
  const int waves = (a.H + 512 * kNC - 1) / (512 * kNC);
  hipLaunchKernelGGL((adaln_sandwich_few_kernel<kNC>), dim3((unsigned)((a.T + a.rows_each - 1) / a.rows_each)), dim3(64 * waves), 0, s, a);
}

template <int NCH>
int launch_many(const SandwichArgs& a, hipStream_t s) {
  constexpr int bytes = 8192 * NCH;  // four fp32 vectors of whole chunks
  static int allowed[64] = {0};
  int dev = 0;
  if (bytes > 60 * 1024 && hipGetDevice(&dev) == hipSuccess && dev >= 0 && (dev >= 64 || allowed[dev] < bytes)) {
    WANMI_REQUIRE(hipFuncSetAttribute(reinterpret_cast<const void*>(&adaln_sandwich_kernel<NCH>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      160 * 1024) == hipSuccess,
                  WANMI_ERR_HIP, "wanmi_adaln_sandwich: %d bytes of LDS refused", bytes);
    if (dev < 64) allowed[dev] = 160 * 1024;
  }
  constexpr int waves = kManyWaves;
  hipLaunchKernelGGL((adaln_sandwich_kernel<NCH>), dim3((unsigned)((a.T + waves - 1) / waves)), dim3(64 * waves), bytes, s, a);
  return check_launch("wanmi_adaln_sandwich");
}

bool aligned16(const void* p) { return ((uintptr_t)p % 16) == 0; }

}  // namespace
}  // namespace wanmi

extern "C" int wanmi_adaln_sandwich(const void* hidden, int64_t ld_hidden, const void* residual, int64_t ld_residual,
                                    const float* post_weight, const float* gate, int64_t ld_gate, const float* mul,
                                    int64_t ld_mul, const float* add, int64_t ld_add, const int32_t* request_ids,
                                    int64_t requests, float residual_scale, int64_t T, int64_t H, float eps, int post_norm,
                                    int norm_type, int quant_type, int zero_rest, void* residual_out, void* out,
                                    uint8_t* scales, void* stream) {
  using namespace wanmi;
  clear_error();
  // (a wave a row: a launch has fewer than 2^32 lanes)
  WANMI_REQUIRE(T >= 0 && T <= (1LL << 26) - 8, WANMI_ERR_ARG, "wanmi_adaln_sandwich: T=%lld must be in [0, 2^26 - 8]", (long long)T);
  WANMI_REQUIRE(H > 0 && H % 32 == 0, WANMI_ERR_ARG, "wanmi_adaln_sandwich: H=%lld must be a positive multiple of 32",
                (long long)H);
  WANMI_REQUIRE(H <= 16384, WANMI_ERR_UNSUPPORTED, "wanmi_adaln_sandwich: H=%lld exceeds 16384", (long long)H);
  for (int n : {post_norm, norm_type})
    WANMI_REQUIRE(n == WANMI_NORM_NONE || n == WANMI_NORM_LAYER || n == WANMI_NORM_RMS, WANMI_ERR_ARG,
                  "wanmi_adaln_sandwich: unknown norm %d", n);
  WANMI_REQUIRE(quant_type == WANMI_QUANT_NONE || quant_type == WANMI_QUANT_MX || quant_type == WANMI_QUANT_ROW, WANMI_ERR_ARG,
                "wanmi_adaln_sandwich: unknown quant_type %d", quant_type);
  WANMI_REQUIRE(eps >= 0.0f, WANMI_ERR_ARG, "wanmi_adaln_sandwich: eps must be >= 0");
  WANMI_REQUIRE(requests >= 0 && requests < (1LL << 31), WANMI_ERR_ARG, "wanmi_adaln_sandwich: requests=%lld out of range",
                (long long)requests);
  WANMI_REQUIRE(request_ids || requests >= 1 || T == 0, WANMI_ERR_ARG, "wanmi_adaln_sandwich: no request to give the rows to");
  if (T == 0) return WANMI_OK;
  WANMI_REQUIRE(hidden && residual_out, WANMI_ERR_ARG, "wanmi_adaln_sandwich: hidden and residual_out must not be null");
  WANMI_REQUIRE(!out || quant_type != WANMI_QUANT_MX || scales, WANMI_ERR_ARG, "wanmi_adaln_sandwich: MX output needs scales");
  for (int64_t ld : {ld_hidden, residual ? ld_residual : ld_hidden})
    WANMI_REQUIRE(ld >= H && ld % 8 == 0, WANMI_ERR_ARG,
                  "wanmi_adaln_sandwich: row strides must be multiples of 8 of at least H, got %lld", (long long)ld);
  for (int64_t ld : {gate ? ld_gate : 0, mul ? ld_mul : 0, add ? ld_add : 0})
    WANMI_REQUIRE(ld == 0 || (ld >= H && ld % 4 == 0), WANMI_ERR_ARG,
                  "wanmi_adaln_sandwich: gate, mul and add rows are a multiple of 4 of at least H apart, or 0, got %lld",
                  (long long)ld);
  for (const void* p : {hidden, residual, (const void*)post_weight, (const void*)gate, (const void*)mul, (const void*)add,
                        (const void*)residual_out, (const void*)out})
    WANMI_REQUIRE(aligned16(p), WANMI_ERR_ARG, "wanmi_adaln_sandwich: tensors must be 16-byte aligned");

  SandwichArgs a;
  a.hidden = static_cast<const uint16_t*>(hidden);
  a.residual = static_cast<const uint16_t*>(residual);
  a.ld_h = ld_hidden;
  a.ld_r = ld_residual;
  a.post_weight = post_weight;
  a.gate = gate;
  a.mul = mul;
  a.add = add;
  a.ld_gate = ld_gate;
  a.ld_mul = ld_mul;
  a.ld_add = ld_add;
  a.ids = request_ids;
  a.requests = (int)requests;
  a.alpha = residual_scale;
  a.eps = eps;
  a.T = T;
  a.H = (int)H;
  a.post_norm = post_norm;
  a.norm = norm_type;
  a.quant = quant_type;
  a.zero_rest = zero_rest;
  a.residual_out = static_cast<uint16_t*>(residual_out);
  a.out = out;
  a.scales = scales;
  hipStream_t s = (hipStream_t)stream;
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  const int nch = (int)((H + 511) / 512);
  if (T <= 2 * cus || nch > 10) {
    // few rows, or more of a row than a wave's registers hold. A workgroup / a wave a row, us: 5120 columns 256 rows 6.4 /
    // 15.8, 512 11.2 / 17.1, 640 16.3 / 17.7, 1024 17.3 / 20.0, 1560 26.3 / 17.1, 4096 46 / 34; 1536 columns 512 rows 5.2 / 6.4,
    // 1024 6.5 / 6.7, 1560 9.0 / 7.4, 4096 15.2 / 13.0 (the bf16 form; MX codes cross at the same places). Past 5120 columns
    // there is the first alone: 7800 rows of 8192 116 us, of 13824 344 (8 bytes a column at 5.5 TB/s: 93 and 157).
    const int waves = H <= 8192 ? nch : (nch + 1) / 2;
    const int64_t resident = (int64_t)cus * (waves <= 10 ? 20 / waves : 1);
    a.rows_each = (T + resident - 1) / resident;
    if (H <= 8192) launch_few<1>(a, s);
    else launch_few<2>(a, s);
    return check_launch("wanmi_adaln_sandwich");
  }
  switch (nch) {
    case 1: return launch_many<1>(a, s);
    case 2: return launch_many<2>(a, s);
    case 3: return launch_many<3>(a, s);
    case 4: return launch_many<4>(a, s);
    case 5: return launch_many<5>(a, s);
    case 6: return launch_many<6>(a, s);
    case 7: return launch_many<7>(a, s);
    case 8: return launch_many<8>(a, s);
    case 9: return launch_many<9>(a, s);
    default: return launch_many<10>(a, s);
  }
}
